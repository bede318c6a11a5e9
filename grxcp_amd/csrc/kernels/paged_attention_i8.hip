// grxDNN attention of one new token per sequence over a paged key-value cache in 8 bits,
// on gfx950.
//
// New: the reference plans attention for grxDNN (ref
// docs/designs/grxcp_roadmap.md:864-877) and ships no code.
//
// The work is divided as over a cache of 16 bits (paged_attention.hip): units of a tile for
// each of a workgroup's four waves, shares of equal size, parts joined in the order of the
// slots. Half the bytes, so a wave's tile has 64 slots where the work is shared, 16 KB of codes
// again. What differs:
//
//  * scores are S^T = K Q^T on the 8-bit matrix cores (v_mfma_i32_16x16x64_i8): the codes of
//    K go in as they lie, with no conversion. A query's row is held as whole numbers of 23
//    bits of its largest value in three digits of base 256 (-128 .. 127), so a product
//    takes three instructions and is exact: what is lost is the rounding of q to 2^-22 of
//    the row's largest value. The slot's scale multiplies the sum;
//  * O^T += V^T P^T on the fp16 matrix cores: the transposing LDS read of bytes brings 8
//    slots of a value's dimension, and a code c becomes fp16 exactly, as the last bits of
//    1024 + (c + 128) less 1152. The weights carry the slots' scales, in units of a power of
//    two that follows the largest of those products (not the largest scale, whose slot may
//    weigh nothing), and are split in two fp16 numbers;
//  * a group of up to 4 (8) query heads leaves 12 (8) of a product's 16 columns empty. They
//    get the same queries again, and each set of columns goes on with a quarter (half) of
//    the tile's slots: the softmax is done once for every score. In the product with V a
//    set's weights of the others' slots are 0, and the sets' results are added at the end;
//  * a lane finds page, row and both scales of one slot of the tile, and hands them to the
//    others through LDS;
//  * K and V go to LDS without registers, 8 lanes to a row of 128 bytes. The products' operands
//    need a row's bytes in four lanes 16 apart, and loads of K in that form straight from
//    memory took the loads' unit four times as long: waves waited to issue in 45 % of their
//    cycles (48 sequences of 33 to 4096 slots 50.6 for 47.7 us, 64 of 20 to 1000 26.6 for
//    21.4). A tile that has come goes to registers whole, and the next one into its place.
//
// us, 32 query and 8 key heads of 128, bf16, a scale for 16 slots: 48 sequences of 33 to 4096
// slots 47.7 (4.3 TB/s; the join 5), 48 of 8000 137 (5.7), 64 of 800 23.7, one of 201 7.0; 2 of
// 131072 with 4 key heads, a scale for each slot, 53 (5.2). What a call has above its bytes
// (6.5 TB/s from one length to the next) are 11 us: launch, lengths, table, queries and the
// first tile one after the other, and the join.

#include "paged_split.h"

#include <cstdio>

namespace grxk {
namespace {

// Slots of a wave's tile: 64, and 32 with two tiles of query heads, for the registers, and where
// a workgroup takes a whole sequence: three of them share a CU then, not two. us, 64 / 32:
// whole sequences, 64 x 8 heads of 800 slots 28.9 / 26.9, 128 x 8 of 800 52.1 / 48.7; shares (three
// or two workgroups to a CU), 48 x 8 of 2000 43.1 / 45.5, 2 x 4 of 131072 51.8 / 53.2.
constexpr int tile_of(int nt, bool whole) { return nt == 1 && !whole ? 64 : 32; }

struct QParams {
  DParams d;                              // pools' strides in 16-byte chunks of codes
  const float* ks; const float* vs;
  int64_t cp, ch, cb;                     // the scales' strides
  PageDiv by_block;
};

// 16-byte chunk of a V row in LDS: chunk ^ vswz(row). The 8 rows of a transposing read (4g ..
// 4g + 3 and 16 + 4g .. 16 + 4g + 3) touch every bank of 128 bytes once.
template <int D> __device__ __forceinline__ int vswz(int row) {
  if constexpr (D == 128) return (row & 3) | (row >> 2 & 4);
  else return (row >> 1 & 1) | (row >> 3 & 2);
}

// The same of a K row: 8 neighbouring rows read at one chunk touch every bank once.
template <int D> __device__ __forceinline__ int kswz(int row) {
  if constexpr (D == 128) return row & 7;
  else return row >> 1 & 3;
}

typedef int i32x2 __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(3))) i32x2* lds_i32x2_t;

// 8 codes as fp16.
__device__ __forceinline__ i32x4 to_half(i32x2 w) {
  typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
  i32x4 r;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t u = (uint32_t)w[i / 2] ^ 0x80808080u;
    const uint32_t h = __builtin_amdgcn_perm(0x64646464u, u, i % 2 ? 0x04030402u : 0x04010400u);
    r[i] = __builtin_bit_cast(int, __builtin_bit_cast(f16x2, h) - f16x2{1152.0f, 1152.0f});
  }
  return r;
}

// 4 values x, |x| scale < 2^22, as whole numbers in digits of base 256: the digits' bytes.
struct Digits { int d[3]; };            // the first is the highest
__device__ __forceinline__ Digits digits4(const float* x, float scale) {
  uint32_t m[4];
#pragma unroll
  for (int i = 0; i < 4; ++i)            // + 1.5 * 2^23 rounds; + 0x8080 makes the lower two unsigned
    m[i] = __float_as_uint(fmaf(x[i], scale, 12582912.0f)) + (0x8080u - 0x400000u);
  const uint32_t a = __builtin_amdgcn_perm(m[1], m[0], 0x05010400u), b = __builtin_amdgcn_perm(m[3], m[2], 0x05010400u);
  const uint32_t c = __builtin_amdgcn_perm(m[1], m[0], 0x0c0c0602u), d = __builtin_amdgcn_perm(m[3], m[2], 0x0c0c0602u);
  return {(int)__builtin_amdgcn_perm(d, c, 0x05040100u), (int)(__builtin_amdgcn_perm(b, a, 0x07060302u) ^ 0x80808080u),
          (int)(__builtin_amdgcn_perm(b, a, 0x05040100u) ^ 0x80808080u)};
}

// Two weights x, y of 0 .. 2^15 as a + b in fp16: 21 bits of each, and nothing below 2^-25. (b may
// be 0, as codes are finite: no product of it needs to show.)
__device__ __forceinline__ void split2(float x, float y, int& a, int& b) {
  typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
  const f16x2 h = __builtin_bit_cast(f16x2, __builtin_amdgcn_cvt_pkrtz(x, y));
  a = __builtin_bit_cast(int, h);
  b = (int)pack_f16x2(x - (float)h[0], y - (float)h[1]);
}

// op over the sets of a group of 16 lanes, in each.
template <int SETS, class Op> __device__ __forceinline__ float over_sets(float v, Op op) {
  if constexpr (SETS >= 2) v = op(v, dpp_f<0x128>(v));   // row_ror 8
  if constexpr (SETS >= 4) v = op(v, dpp_f<0x124>(v));   // row_ror 4
  return v;
}

template <AttnType T> __device__ __forceinline__ void unpack8(u32x4 w, float* f) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (T == AttnType::BF16) {
      f[2 * i] = __uint_as_float(w[i] << 16);
      f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    } else {
      f[2 * i] = f16_to_f32((uint16_t)w[i]);
      f[2 * i + 1] = f16_to_f32((uint16_t)(w[i] >> 16));
    }
  }
}

template <AttnType T, int D, int NT, int SETS, int kTile, bool ONCE>
__global__ __launch_bounds__(64 * kWaves, NT == 1 && kTile == 32 ? 3 : 2) void decode_split_i8(QParams qp) {
  using W = PIo<AttnType::F16>;      // the weights' type
  constexpr float kUnscale = 0x1p-11f;
  static_assert(W::kTop == 11.0f);
  const DParams& p = qp.d;
  constexpr int F = D / 64;          // contraction steps of a score
  constexpr int DT = D / 16;         // tiles of the head dimension
  constexpr int CH = D / 16;         // chunks of a row
  constexpr int RPI = 64 / CH;       // V rows per load
  constexpr int KT = kTile / 16;     // tiles of 16 slots
  constexpr int HC = 16 / SETS;      // columns of a set: query heads
  constexpr int MT = KT / SETS;      // tiles of 16 slots that a lane looks after
  static_assert(NT == 1 || SETS == 1, "sets are for groups that leave columns empty");
  constexpr int kStage = kTile * CH; // chunks of a tile of K or V
  constexpr int kPitch = D + 4;
  constexpr int kV = kWaves * 2 * kStage * 16, kMerge = kWaves * 16 * kPitch * 4;
  __shared__ __attribute__((aligned(1024))) uint8_t smem[kV > kMerge ? kV : kMerge];
  __shared__ uint64_t rows[kWaves][2][kTile];
  __shared__ __attribute__((aligned(16))) float scales[kWaves][2][kTile];
  __shared__ float ml[kWaves][2][16];

  const int tid = threadIdx.x, lane = tid & 63, l16 = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int set = l16 / HC;

  uint32_t b, it, i, share, left;
  int len64;
  if (!find_share(p, lane, b, it, i, share, left, len64)) return;

  uint8_t* ktile = smem + wave * 2 * kStage * 16;
  uint8_t* vtile = ktile + kStage * 16;
  const int of = kWaves / p.hw;      // waves of a key head
  const int hd = wave / of, sub = wave - hd * of;

  while (left > 0) {
    const int len = b < 64 ? __builtin_amdgcn_readlane(len64, b)
                           : __builtin_amdgcn_readfirstlane(clamp_length(p.view.lengths[b], p.view.room));
    const uint32_t n = units_of(p, len);
    if (p.whole) left = n;
    const uint32_t take = min(left, n - i);
    const int hg = (int)it / p.gtiles, q0 = ((int)it - hg * p.gtiles) * 16 * NT;   // first query head of the group
    const int h = hg * p.hw + hd;                                       // the wave's key head
    const int* table = p.view.table + (int64_t)b * p.view.table_rs;
    const uint8_t* kbase = p.k + 16ull * h * p.k_sh;
    const uint8_t* vbase = p.v + 16ull * h * p.v_sh;

    f32x4 o[NT][DT];
    float m[NT], l[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      m[t] = -INFINITY;              // no slot yet
      l[t] = 0.0f;
#pragma unroll
      for (int d = 0; d < DT; ++d) o[t][d] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    }
    // A slot's product of weight and scale is held in units of 2^unit_o: the largest so far is 2^11
    // .. 2^15 of them, whatever larger scales the slots without weight have. m is a whole number:
    // where it rises, the weights' unit falls by a power of two, and o stays as it is.
    int unit_o[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) unit_o[t] = -4096;

    float ksr, vsr;                  // the scales of the lane's slot
    uint64_t live;                   // the tile's slots that are there
    const int step = 1 << p.shift;
    int key = (int)(i << p.shift) + sub * kTile;                        // the wave's first slot
    const int end = (int)min((uint32_t)len, (i + take) << p.shift);
    auto entry = [&](int key0) __attribute__((always_inline)) {
      const int j = key0 + lane;
      return lane < kTile && j < end ? table[div_page(p.view.div, j)] : -1;
    };
    // Loads of the tile at key0, whose table entries are e.
    auto issue = [&](int key0, int e) __attribute__((always_inline)) {
      const int j = key0 + lane;
      const int page = lane < kTile && j < end ? checked_page(e, p.view.pages) : -1;
      const int row = j - div_page(p.view.div, j) * p.view.page;
      const bool there = page >= 0;
      const uint64_t pg = (uint32_t)page, r64 = (uint32_t)row;
      if (lane < kTile) {
        rows[wave][0][lane] = (uint64_t)(there ? kbase + 16 * (pg * p.k_sp + r64 * p.k_ss) : (const uint8_t*)zero_row);
        rows[wave][1][lane] = (uint64_t)(there ? vbase + 16 * (pg * p.v_sp + r64 * p.v_ss) : (const uint8_t*)zero_row);
      }
      live = __ballot(there);
      ksr = vsr = 0.0f;
      if (there) {
        const int64_t at = page * qp.cp + h * qp.ch + div_page(qp.by_block, row) * qp.cb;
        ksr = qp.ks[at];
        vsr = qp.vs[at];
      }
      wave_fence();
#pragma unroll
      for (int x = 0; x < kTile / RPI; ++x) {
        const int r = RPI * x + lane / CH;
        dma16<ONCE>((const uint8_t*)rows[wave][0][r] + 16 * ((lane % CH) ^ kswz<D>(r)), lds_addr(ktile + 1024 * x));
      }
#pragma unroll
      for (int x = 0; x < kTile / RPI; ++x) {
        const int r = RPI * x + lane / CH;
        dma16<ONCE>((const uint8_t*)rows[wave][1][r] + 16 * ((lane % CH) ^ vswz<D>(r)), lds_addr(vtile + 1024 * x));
      }
    };
    int e = entry(key);
    int next = entry(key + step);

    u32x4 raw[NT][F][2];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const int r = q0 + 16 * t + (l16 & (HC - 1));
      const uint8_t* src = r < p.group ? p.q + (int64_t)b * p.q_sb + (h * p.group + r) * p.q_sh : (const uint8_t*)zero_row;
#pragma unroll
      for (int f = 0; f < F; ++f)
#pragma unroll
        for (int x = 0; x < 2; ++x) raw[t][f][x] = *(const u32x4*)(src + 2 * (64 * f + 16 * g + 8 * x));
    }
    issue(key, e);                   // (zeros where the wave has no slot)
    // The queries' digits, and what a sum of them stands for.
    i32x4 qd[NT][3][F];
    float unit[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      float top = 0.0f, odd = 0.0f;
#pragma unroll
      for (int f = 0; f < F; ++f)
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          float v[8];
          unpack8<T>(raw[t][f][x], v);
#pragma unroll
          for (int u = 0; u < 8; ++u) {
            top = fmaxf(top, fabsf(v[u]));
            odd = fmaf(v[u], 0.0f, odd);         // NaN where a value is not finite
          }
        }
      top = over_query(top, [](float a, float x) { return fmaxf(a, x); });
      odd = over_query(odd, [](float a, float x) { return a + x; });
      // 2^e <= top < 2^(e+1): top * 2^(21-e) is below 2^22
      const int e = min(max((int)(__float_as_uint(top) >> 23), 127 - 105), 254) - 127;
      const float scale = __uint_as_float((uint32_t)(127 + 21 - e) << 23);
      unit[t] = __uint_as_float((uint32_t)(127 - 21 + e) << 23) * p.c + odd;
#pragma unroll
      for (int f = 0; f < F; ++f)
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          float v[8];
          unpack8<T>(raw[t][f][x / 2], v);
          const Digits q = digits4(v + x % 2 * 4, scale);
#pragma unroll
          for (int y = 0; y < 3; ++y) qd[t][y][f][x] = q.d[y];
        }
    }

    while (key < end) {
      wait_all();
      const uint64_t mask = live;
      if (lane < kTile) {
        scales[wave][0][lane] = ksr;
        scales[wave][1][lane] = vsr;
      }
      wave_fence();
      // The tile into registers; then its place takes the next one.
      i32x4 kf[KT][F];
#pragma unroll
      for (int kt = 0; kt < KT; ++kt)
#pragma unroll
        for (int f = 0; f < F; ++f) {
          const int r = 16 * kt + l16;
          kf[kt][f] = *(const i32x4*)(ktile + r * D + 16 * ((4 * f + g) ^ kswz<D>(r)));
        }
      i32x2 vc[DT][KT / 2];
      const int in = l16 >> 1;                   // the lane's row of a transposing read
      const int r0 = in < 4 ? 4 * g + in : 12 + 4 * g + in;
#pragma unroll
      for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int x = 0; x < KT / 2; ++x) {
          const int r = 32 * x + r0;
          vc[d][x] = __builtin_amdgcn_ds_read_tr8_b64_v2i32(
              (lds_i32x2_t)(vtile + r * D + 16 * (d ^ vswz<D>(r)) + 8 * (lane & 1)));
        }
      if (key + step < end) {
        asm volatile("" ::: "memory");
        __builtin_amdgcn_s_waitcnt(0xc07f);      // lgkmcnt(0): the reads are done
        asm volatile("" ::: "memory");
        issue(key + step, next);
        next = entry(key + 2 * step);
      }
      key += step;
      if (!mask) continue;                       // nothing to add
      i32x4 pf[NT][KT / 2], pr[NT][KT / 2];      // the weights: leading bits, rest
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        f32x4 s[MT];                             // of the lane's tiles, set * MT ..
#pragma unroll
        for (int k = 0; k < MT; ++k) {
          i32x4 a[3];
#pragma unroll
          for (int x = 0; x < 3; ++x) {
#pragma unroll
            for (int c = 0; c < SETS; ++c) {
              i32x4 sum = {0, 0, 0, 0};
#pragma unroll
              for (int f = 0; f < F; ++f)
                sum = __builtin_amdgcn_mfma_i32_16x16x64_i8(kf[c * MT + k][f], qd[t][x][f], sum, 0, 0, 0);
              if (c == 0) a[x] = sum;
              else
#pragma unroll
                for (int r = 0; r < 4; ++r) a[x][r] = set == c ? sum[r] : a[x][r];
            }
          }
          const f32x4 by = *(const f32x4*)&scales[wave][0][16 * (set * MT + k) + 4 * g];
#pragma unroll
          for (int r = 0; r < 4; ++r)
            s[k][r] = fmaf(fmaf((float)a[0][r], 256.0f, (float)a[1][r]), 256.0f, (float)a[2][r]) * (by[r] * unit[t]);
        }
        if (mask != (kTile == 64 ? ~0ull : 0xffffffffull)) {
          const uint64_t mine = mask >> (16 * set * MT + 4 * g);
#pragma unroll
          for (int k = 0; k < MT; ++k)
#pragma unroll
            for (int r = 0; r < 4; ++r)
              if (!(mine >> (16 * k + r) & 1)) s[k][r] = -INFINITY;
        }
        float mx = s[0][0];
#pragma unroll
        for (int x = 1; x < 4 * MT; ++x) mx = fmaxf(mx, s[x / 4][x % 4]);
        mx = over_sets<SETS>(mx, [](float a, float x) { return fmaxf(a, x); });
        mx = over_query(mx, [](float a, float x) { return fmaxf(a, x); });
        mx = fmaxf(mx, kLowest);     // -inf scores weigh 0; a row of only such has l = 0 and is NaN
        const bool raise = mx - m[t] > kLazy;
        if (__ballot(raise)) {
          const float top = raise ? ceilf(mx) : m[t], drop = raise ? m[t] - top : 0.0f;
          m[t] = top;
          l[t] *= __builtin_amdgcn_exp2f(drop);
          unit_o[t] = max(unit_o[t] + (int)fmaxf(drop, -1024.0f), -4096);
        }
        float most = 0.0f;
#pragma unroll
        for (int k = 0; k < MT; ++k) {
          const f32x4 by = *(const f32x4*)&scales[wave][1][16 * (set * MT + k) + 4 * g];
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const float w = __builtin_amdgcn_exp2f((s[k][r] - m[t]) + W::kTop);
            l[t] += w;
            s[k][r] = w * by[r];
            most = fmaxf(most, s[k][r]);
          }
        }
        if (__ballot(most > ldexpf(0x1p15f, unit_o[t]))) {
          most = over_sets<SETS>(most, [](float a, float x) { return fmaxf(a, x); });
          most = over_query(most, [](float a, float x) { return fmaxf(a, x); });
          const int up = max(unit_o[t], (int)(__float_as_uint(most) >> 23) - 127 - 11);
          const float f = ldexpf(1.0f, unit_o[t] - up);
          unit_o[t] = up;
#pragma unroll
          for (int d = 0; d < DT; ++d) o[t][d] *= f;
        }
        int hi[MT][2], lo[MT][2];
#pragma unroll
        for (int k = 0; k < MT; ++k)
#pragma unroll
          for (int x = 0; x < 2; ++x)
            split2(ldexpf(s[k][2 * x], -unit_o[t]), ldexpf(s[k][2 * x + 1], -unit_o[t]), hi[k][x], lo[k][x]);
#pragma unroll
        for (int kt = 0; kt < KT; ++kt)
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            const bool own = SETS == 1 || set == kt / MT;
            pf[t][kt / 2][kt % 2 * 2 + x] = own ? hi[kt % MT][x] : 0;
            pr[t][kt / 2][kt % 2 * 2 + x] = own ? lo[kt % MT][x] : 0;
          }
      }
#pragma unroll
      for (int d = 0; d < DT; ++d) {
        i32x4 vf[KT / 2];
#pragma unroll
        for (int x = 0; x < KT / 2; ++x) vf[x] = to_half(vc[d][x]);
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int x = 0; x < KT / 2; ++x) o[t][d] = W::mma(vf[x], pf[t][x], o[t][d]);
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int x = 0; x < KT / 2; ++x) o[t][d] = W::mma(vf[x], pr[t][x], o[t][d]);
      }
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
      for (int d = 0; d < DT; ++d) {
        f32x4 x;
#pragma unroll
        for (int r = 0; r < 4; ++r)
          x[r] = over_sets<SETS>(ldexpf(o[t][d][r], unit_o[t] - 11), [](float a, float y) { return a + y; });
        *(f32x4*)&mo[(wave * 16 + l16) * kPitch + 16 * d + 4 * g] = x;
      }
      const float sum = over_query(over_sets<SETS>(l[t], [](float a, float x) { return a + x; }),
                                   [](float a, float x) { return a + x; }) * kUnscale;
      if (g == 0) {
        ml[wave][0][l16] = m[t];
        ml[wave][1][l16] = sum;
      }
      __syncthreads();
      meet<T, D>(p, tid, of, hg, q0, 16 * t, b, part, whole, mo, ml);
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

// ---- launch --------------------------------------------------------------------

Plan plan_of(int B, int H, int heads, int D, int W, int page, bool neighbours) {
  Plan x{};
  const int group = H / heads;
  x.nt = group > 16 ? 2 : 1;
  x.gtiles = (group + 16 * x.nt - 1) / (16 * x.nt);
  x.rows = std::min(group, 16 * x.nt);
  x.room = (int64_t)W * page;
  x.slots = (x.room + 255) / 256 * 256;
  const int64_t each = (int64_t)B * heads * x.gtiles;
  // A workgroup per (sequence, head) and no join where no sequence is long: up to 512 slots
  // always, up to 1024 where those workgroups go evenly on the CUs. us, split and joined /
  // whole: 8 heads of one sequence of 500 slots 11.7 / 9.5, of 8 sequences
  // 12.4 / 11.5; 32 x 8 heads of 1000 23.4 / 19.5, 64 x 8 of 800 35.8 / 28.8, of 20 to 1000
  // 31.1 / 28.8, but 16 x 8 of 1000 16.9 / 17.7, 48 x 8 of 1000 30.3 / 32.3.
  const int cus = compute_units();
  const bool even = each >= cus && (each % cus == 0 || each >= 4 * cus);
  x.whole = (x.room <= 512 || (x.room <= 1024 && even)) && each <= (1 << 20);
  x.hw = 1;
  if (!x.whole && neighbours)
    for (int hw = 4; hw > 1 && x.hw == 1; hw /= 2)
      if (heads % hw == 0 && (int64_t)B * (heads / hw) * x.gtiles >= 64) x.hw = hw;
  x.items = (int64_t)B * (heads / x.hw) * x.gtiles;
  x.wgs = x.whole ? (int)x.items : 2 * cus;
  const size_t parts = x.whole ? (size_t)x.items : (size_t)x.items + x.wgs;
  if (!x.whole) x.ml = (parts * x.hw * x.rows * 2 + 3) / 4 * 4;
  if (!x.whole) x.po = parts * x.hw * x.rows * D;
  return x;
}

template <AttnType T, int D>
hipError_t run(const PagedAttnDesc& d, const QuantScales& q, hipStream_t s) {
  const Plan x = plan_of(d.c.B, d.H, d.c.heads, D, d.c.W, d.c.page, neighbours(d.c.k_sh, d.c.k_ss));
  QParams qp{};
  DParams& p = qp.d;
  p.view = {d.c.table, d.c.table_rs, d.c.lengths, d.c.pages, d.c.page, d.c.W * d.c.page, page_div(d.c.page)};
  p.k = (const uint8_t*)d.c.k; p.k_sp = d.c.k_sp / 16; p.k_sh = d.c.k_sh / 16; p.k_ss = d.c.k_ss / 16;
  p.v = (const uint8_t*)d.c.v; p.v_sp = d.c.v_sp / 16; p.v_sh = d.c.v_sh / 16; p.v_ss = d.c.v_ss / 16;
  p.q = (const uint8_t*)d.q; p.q_sb = 2 * d.q_sb; p.q_sh = 2 * d.q_sh;
  p.o = (uint8_t*)d.o; p.o_sb = 2 * d.o_sb; p.o_sh = 2 * d.o_sh;
  float* ws = (float*)d.ws;
  p.ml = ws;
  p.po = ws + x.ml;
  p.slots = x.slots;
  p.B = d.c.B; p.H = d.H; p.heads = d.c.heads; p.group = d.H / d.c.heads;
  p.hw = x.hw; p.shift = (tile_of(x.nt, x.whole) == 64 ? 6 : 5) + (x.hw == 4 ? 0 : x.hw == 2 ? 1 : 2);
  p.gtiles = x.gtiles; p.items = d.c.heads / x.hw * x.gtiles; p.rows = x.rows; p.wgs = x.wgs; p.whole = x.whole;
  p.c = d.scale * 1.4426950408889634f;
  qp.ks = q.k; qp.vs = q.v;
  qp.cp = q.sp; qp.ch = q.sh; qp.cb = q.sb;
  qp.by_block = page_div(q.block);
  if (log_dnn_launches())
    std::fprintf(stderr, "grxdnn: paged attention i8 %s b=%d h=%d hkv=%d d=%d page=%d block=%d room=%d kernel=%s%d\n",
                 T == AttnType::BF16 ? "bf16" : "f16", p.B, p.H, p.heads, D, p.view.page, q.block, p.view.room,
                 x.whole ? "whole" : "split", x.hw);
  const dim3 grid(x.wgs), threads(64 * kWaves);
  auto go = [&](auto kern) { hipLaunchKernelGGL(kern, grid, threads, 0, s, qp); };
  if (x.nt == 2) {
    if (x.gtiles == 1) go(decode_split_i8<T, D, 2, 1, 32, true>);
    else go(decode_split_i8<T, D, 2, 1, 32, false>);
  } else if (x.whole) {
    if (p.group <= 8) go(decode_split_i8<T, D, 1, 2, 32, true>);
    else go(decode_split_i8<T, D, 1, 1, 32, true>);
  } else {
    if (p.group <= 4) go(decode_split_i8<T, D, 1, 4, 64, true>);
    else if (p.group <= 8) go(decode_split_i8<T, D, 1, 2, 64, true>);
    else go(decode_split_i8<T, D, 1, 1, 64, true>);
  }
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess || x.whole) return e;
  const JoinPlan j = join_plan(x, p.B, p.H, p.heads, false);
  hipLaunchKernelGGL((decode_join<T, D>), dim3((unsigned)j.jobs, (unsigned)std::min(p.B, 65535)), dim3(256), 0, s, p,
                     (uint32_t)j.outs, j.apiece, (uint32_t)j.chunks);
  return hipGetLastError();
}

}  // namespace

size_t paged_attention_i8_workspace(const PagedCache& c, int H) {
  const Plan x = plan_of(c.B, H, c.heads, c.D, c.W, c.page, neighbours(c.k_sh, c.k_ss));
  return (x.ml + x.po) * sizeof(float);
}

bool paged_attention_i8_fits(const PagedCache& c, int H) {
  const Plan x = plan_of(c.B, H, c.heads, c.D, c.W, c.page, neighbours(c.k_sh, c.k_ss));
  return (double)x.items * (x.slots / 32) < 0x1p31 &&
         join_plan(x, c.B, H, c.heads, false).jobs <= max_workgroups(256);
}

hipError_t launch_paged_attention_i8(AttnType t, const PagedAttnDesc& d, const QuantScales& q, hipStream_t s) {
  if (t == AttnType::BF16) {
    if (d.c.D == 128) return run<AttnType::BF16, 128>(d, q, s);
    if (d.c.D == 64) return run<AttnType::BF16, 64>(d, q, s);
  } else {
    if (d.c.D == 128) return run<AttnType::F16, 128>(d, q, s);
    if (d.c.D == 64) return run<AttnType::F16, 64>(d, q, s);
  }
  return hipErrorNotSupported;
}

}  // namespace grxk
