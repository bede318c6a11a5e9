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

#include "paged_split.h"

#include <cstdio>

namespace grxk {
namespace {

constexpr int kTile = 32;                 // slots of a wave's tile

// Workgroups that share a CU: registers (D = 64 has half the accumulators) and LDS. us at
// D = 64, three / four (28 bytes of registers spilled, shares a quarter shorter): 24 x 16
// heads of 500 to 3001 slots with weights 42.3 / 50.8, 16 x 16 of 8192 94.6 / 103.4; with two
// tiles of query heads, two / three: 32 x 2 of 4000 23.1 / 26.4.
template <int D, int NT> constexpr int wgs_per_cu() { return D == 64 && NT == 1 ? 3 : 2; }

// ---- the split -----------------------------------------------------------------

// 16-byte chunk of a V row in LDS: chunk ^ vswz(row).
template <int D> __device__ __forceinline__ int vswz(int row) {
  if constexpr (D == 128) return 2 * (row & 7);
  else return 2 * ((row >> 1) & 3);
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

  uint32_t b, it, i, share, left;
  int len64;
  if (!find_share(p, lane, b, it, i, share, left, len64)) return;

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
