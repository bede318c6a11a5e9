// grxDNN log probabilities of given tokens over rows of logits, with entropy and
// the top alternatives, and their gradient in the logits, on gfx950.
//
// New: the reference plans softmax for grxDNN (ref
// docs/designs/grxcp_roadmap.md:864-877) and ships no code.
//
// Forward: one pass over the logits. A row, or a piece of it where rows are few, goes
// to a wave; every lane keeps
//   s = sum 2^(x log2 e - r),  t = sum 2^(x log2 e - r) (x log2 e - r)
// over its elements with a reference r of its own that moves only when a batch's
// maximum exceeds it by more than 8, so an element costs an unpack, half a max, two
// fmas, an add and an exp2: the exp2 (a quarter rate instruction) makes that 8.5
// lane operations against the 64 a CU does in a cycle, which is 8 TB/s of bf16, little
// above what the memory gives. Then log sum exp = max + log S and entropy =
// log S - T / S from the sums moved to the row's maximum.
// x log2 e - r is one fma: off by half a step of itself. What the rounded log2 e is off by
// and what r is cancel when the sums move to the maximum, as 2^(r - max log2 e) takes the
// same two numbers: an element is off by 2^-26 |x - max| for it, whatever |x| is. A row
// whose maximum is outside -64 .. 64, far within where r stays harmless, or whose sums are
// not finite, is read again with x - max formed first. As e^0 is among them, S is at least
// 1 and T at most 0: held to that, no probability is above 1 and no entropy below 0.
//
// Alternatives: the same pass compares each batch's maximum with a threshold that K
// elements already read reach, and only where it is higher looks at the elements: those
// from it on go to a list in LDS. The first threshold is the K-th
// largest of the 128 maxima of the wave's lanes' half batches; it is raised after batches
// 2, 4, 8, ... to the list's K-th largest, so a wave lists about K of every doubling of
// what it has read. Elements are ranked by value, then by lower index; as batches come in
// index order an equal value in a later batch never outranks one in the list. A batch with
// more such elements than that (a row that rises, a vocabulary mask's run of -inf) sets the
// threshold from its own maxima again and lists, of what equals it, only the first few: us
// of 2048 x 32000 bf16 with 8 alternatives, 39 in no order, 51 where all but 5 are -inf,
// 110 rising. What no such step fits (NaN, +inf, a last batch that rises by hundreds) takes
// the direct way: the largest element below the last one, K times.
//
// Backward: one element-wise pass, bound by reading x and writing dx.
//
// us: 32 rows of 131072 bf16 with 8 alternatives 14.3 (8.4 MB: two launches, 10 and 4; in
// the first the VALU is at work half of the time, at five times the instructions that the
// sums take), 256 rows 30.4 (2.2 TB/s; 17 of it VALU work), 2048 x 32000 without any 25.2
// (5.2), 4096 x 32001 fp32 86 (6.1); the gradient of 8192 x 65536 bf16 with entropy 346
// (6.2), of 500 x 50001 fp16 21.3 and of 500 x 50000 20.3 (4.7, 4.9).

#include "../launch.h"
#include "device_common.h"
#include "paged_common.h"
#include "row_io.h"

#include <algorithm>
#include <climits>

namespace grxk {
namespace {

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr float kLowest = -__FLT_MAX__;
constexpr int kU = 4;         // chunks of a thread (backward, and a forward batch of a whole row)
constexpr int kMaxTop = 64;
constexpr int kMaxPieces = 64, kMaxKeys = 1024;   // of a row, and what they list

struct LParams {
  const uint8_t* x;
  int64_t x_rs, rows;
  int vocab, top;
  int align_mask;      // RowChunks
  int pieces, each;    // pieces of a row, chunks of a piece
  const int* tokens;
  float* logprob; float* lse; float* entropy;
  float* top_logprob; int* top_index;
  float* sums;         // [rows, pieces, 4]: maximum, S, T relative to it
  uint64_t* keys;      // [rows, pieces, top], largest first
};

// A value and its place as one number: larger values first, of equal ones the
// lower place. Zero is below every key.
__device__ __forceinline__ uint64_t rank_key(float v, int j) {
  return (uint64_t)order_key(__float_as_uint(v)) << 32 | (uint32_t)~j;
}
__device__ __forceinline__ int key_place(uint64_t k) { return (int)~(uint32_t)k; }
__device__ __forceinline__ float key_value(uint64_t k) {
  const uint32_t u = (uint32_t)(k >> 32);
  if (u == 0xffffffffu) return __uint_as_float(0x7fc00000u);
  return __uint_as_float((u & 0x80000000u) ? u & 0x7fffffffu : ~u);
}

// Sums of a row or a part of it, relative to its maximum m (kept finite, so that a
// row of only -inf has S = 0): S = sum e^(x - m), T = sum e^(x - m) (x - m).
struct Sums {
  float m, s, t;
};
// The same relative to m >= v.m. A part without a sum stays without one.
__device__ __forceinline__ Sums moved(Sums v, float m) {
  const float d = v.m - m, f = __builtin_amdgcn_exp2f(d * kLog2e);
  const float t = fmaf(v.s, d, v.t);
  return {m, v.s * f, v.s == 0.0f || f == 0.0f ? 0.0f : t * f};
}

// Number of the first c keys that are larger than k. The list is read two keys at a
// time; what lies behind its end (up to a multiple of 8) is not counted.
typedef unsigned long long u64x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ int rank_of(const uint64_t* keys, int c, uint64_t k) {
  int r = 0;
  for (int i = 0; i < c; i += 8) {
    u64x2 w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) w[j] = ((const u64x2*)keys)[i / 2 + j];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      r += i + 2 * j < c && w[j][0] > k;
      r += i + 2 * j + 1 < c && w[j][1] > k;
    }
  }
  return r;
}

// The largest key that K of the wave's keys reach, N of them to a lane, or one below it
// that no more than these reach: bit by bit from the top, as far down as keys of T differ
// (the rest is 0, or all ones below the keys of 0). 0 if there are fewer than K above 0.
template <NormType T, int N> __device__ __forceinline__ uint32_t reached_by(const uint32_t (&key)[N], int K) {
  constexpr int kLast = T == NormType::F32 ? 0 : T == NormType::BF16 ? 16 : 13;
  uint32_t v = 0;
  for (int bit = 31; bit >= kLast; --bit) {
    const uint32_t t = v | (1u << bit);
    int c = 0;
#pragma unroll
    for (int q = 0; q < N; ++q) c += __popcll(__ballot(key[q] >= t));
    if (c >= K) v = t;
    if (c == K) break;
  }
  return v && v < 0x80000000u ? v | ((1u << kLast) - 1) : v;
}
// A bound's value; -inf for what is below every value.
__device__ __forceinline__ float bound_value(uint32_t key) {
  return key <= 0x007fffffu ? -INFINITY : key_value((uint64_t)key << 32);
}
// The next value above x (x is no NaN): of -0 as of 0.
__device__ __forceinline__ float above(float x) {
  const uint32_t u = order_key(__float_as_uint(x));
  return x == INFINITY ? x : key_value((uint64_t)(u + 1) << 32);
}

// The list of a wave. A row may list all of its elements where it has fewer than K for
// every lane.
constexpr int kCap = 512;
struct Shared {
  __attribute__((aligned(16))) uint64_t list[kCap];
  uint64_t best[kMaxTop];
};

// Of a list of c <= 64 N keys what reaches the bound that K of them reach; returns that
// bound.
template <NormType T, int N>
__device__ __forceinline__ uint32_t refine(uint64_t* list, int& c, int top) {
  const int lane = threadIdx.x;
  uint64_t key[N];
  uint32_t hi[N];
#pragma unroll
  for (int q = 0; q < N; ++q) {
    key[q] = 64 * q + lane < c ? list[64 * q + lane] : 0;
    hi[q] = (uint32_t)(key[q] >> 32);
  }
  const uint32_t bound = max(reached_by<T>(hi, top), 1u);
  int to = 0;
#pragma unroll
  for (int q = 0; q < N; ++q) {
    const uint64_t stay = __ballot(hi[q] >= bound);
    if (hi[q] >= bound)
      list[to + (int)__builtin_amdgcn_mbcnt_hi((uint32_t)(stay >> 32),
                                               __builtin_amdgcn_mbcnt_lo((uint32_t)stay, 0))] = key[q];
    to += __popcll(stay);
  }
  c = to;
  return bound;
}
template <NormType T>
__device__ __forceinline__ uint32_t refine_list(uint64_t* list, int& c, int top) {
  return c <= 64 ? refine<T, 1>(list, c, top) : refine<T, kCap / 64>(list, c, top);
}

// Of a list of c keys what reaches `bound`.
__device__ __forceinline__ void keep(uint64_t* list, int& c, uint32_t bound) {
  int to = 0;
#pragma unroll 1
  for (int i = 0; i < c; i += 64) {
    const uint64_t key = i + (int)threadIdx.x < c ? list[i + threadIdx.x] : 0;
    const bool stay = (uint32_t)(key >> 32) >= bound;
    const uint64_t all = __ballot(stay);
    if (stay)
      list[to + (int)__builtin_amdgcn_mbcnt_hi((uint32_t)(all >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)all, 0))] = key;
    to += __popcll(all);
  }
  c = to;
}

// The K largest of a list of c keys, in order in `best`. Returns how many there are.
template <NormType T>
__device__ __forceinline__ int finish(Shared& sh, int top, int c) {
  if (c > 64) refine_list<T>(sh.list, c, top);   // (a short list is ranked as it is)
  __builtin_amdgcn_wave_barrier();
  for (int i = threadIdx.x; i < c; i += 64) {
    const uint64_t k = sh.list[i];
    const int r = rank_of(sh.list, c, k);
    if (r < top) sh.best[r] = k;
  }
  __builtin_amdgcn_wave_barrier();
  return min(c, top);
}

// One row, or a piece of one, per wave.
template <NormType T, bool AL, bool TOP>
__global__ __launch_bounds__(64, AL ? 4 : 3) void logprob_pieces(LParams p) {
  using IO = Io<T>;
  constexpr int V = IO::kVec, NT = 64, U = kU;
  constexpr uint32_t kNone = T == NormType::F32 ? 0xff800000u : T == NormType::BF16 ? 0xff80ff80u : 0xfc00fc00u;
  const u32x4 none = {kNone, kNone, kNone, kNone};     // -inf: outside the row
  __shared__ Shared sh;
  const int tid = threadIdx.x;
  const int64_t jobs = p.rows * p.pieces;
  for (int64_t job = blockIdx.x; job < jobs; job += gridDim.x) {
    // (pieces: of fewer than 2048 rows)
    const int64_t row = p.pieces == 1 ? job : (uint32_t)job / (uint32_t)p.pieces;
    const int piece = p.pieces == 1 ? 0 : (int)(job - row * p.pieces);
    const uint8_t* x = p.x + row * p.x_rs * (int64_t)(16 / V);
    const RowChunks<T, AL> rc(x, p.vocab, p.align_mask);
    const int c0 = piece * p.each, c1 = p.pieces == 1 ? INT_MAX : c0 + p.each;
    auto load = [&](int c) __attribute__((always_inline)) { return c < c1 && rc.any(c) ? rc.load(x, c, none) : none; };
    // Places of chunk c that are in the row and the piece.
    auto has = [&](int c, int e) __attribute__((always_inline)) { return c < c1 && rc.any(c) && rc.has(c, e); };

    // Only the packed batch stays in registers between the passes over it.
    auto hold = [&](u32x4 (&w)[U]) __attribute__((always_inline)) {
#pragma unroll
      for (int q = 0; q < U; ++q) asm volatile("" : "+v"(w[q]));
    };
    int listed = 0;                            // keys on the wave's list
    float m = -INFINITY, r = -1000.0f, s = 0.0f, t = 0.0f;
    float limit = -INFINITY;                   // the wave's: values from it on may be alternatives
    bool over = false;                         // the list lost some
    u32x4 raw[U];
#pragma unroll
    for (int q = 0; q < U; ++q) raw[q] = load(c0 + tid + NT * q);
    for (int c = c0 + tid, batch = 0;; c += U * NT, ++batch) {
      u32x4 cur[U];
#pragma unroll
      for (int q = 0; q < U; ++q) cur[q] = raw[q];
      // (uniform: the first thread's next chunk)
      const int next = c - tid + U * NT;
      const bool more = next < c1 && rc.any(next);
      if (more)
#pragma unroll
        for (int q = 0; q < U; ++q) raw[q] = load(c + (U + q) * NT);
      float high[U];
#pragma unroll
      for (int q = 0; q < U; ++q) {
        float v[V];
        IO::unpack(cur[q], v);
        high[q] = v[0];
#pragma unroll
        for (int e = 1; e < V; ++e) high[q] = fmaxf(high[q], v[e]);
      }
      float top = high[0];
#pragma unroll
      for (int q = 1; q < U; ++q) top = fmaxf(top, high[q]);
      m = fmaxf(m, top);
      const float top2 = top * kLog2e;
      if (top2 > r + 8.0f) {
        const float f = __builtin_amdgcn_exp2f(r - top2);
        t = f * fmaf(s, r - top2, t);
        s *= f;
        r = top2;
      }
      hold(cur);
      float bs = 0.0f, bt = 0.0f;
#pragma unroll
      for (int q = 0; q < U; ++q) {
        float v[V];
        IO::unpack(cur[q], v);
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const float d = fmaf(v[e], kLog2e, -r), w = __builtin_amdgcn_exp2f(d);
          bs += w;
          bt = fmaf(w, d, bt);
        }
      }
      if (__ballot(bt != bt)) {                // -inf among them: 0 * -inf stands for 0
        hold(cur);
        bt = 0.0f;
#pragma unroll 1
        for (int q = 0; q < U; ++q) {
          float v[V];
          IO::unpack(cur[0], v);
#pragma unroll
          for (int e = 0; e < V; ++e) {
            const float d = fmaf(v[e], kLog2e, -r), w = __builtin_amdgcn_exp2f(d);
            bt += w == 0.0f ? 0.0f : w * d;
          }
          const u32x4 w = cur[0];
#pragma unroll
          for (int u = 0; u + 1 < U; ++u) cur[u] = cur[u + 1];
          cur[U - 1] = w;
        }
      }
      s += bs;
      t += bt;
      if constexpr (TOP) {
        // What K of the batch's elements reach: the K-th largest of its parts' maxima. Parts
        // of two chunks a lane where fewer than K of them fit the list.
        auto reach = [&]() __attribute__((always_inline)) {
          if ((kMaxTop - 1) * 2 * V <= kCap || p.top <= kCap / (2 * V)) {
            const uint32_t key[2] = {order_key(__float_as_uint(fmaxf(high[0], high[1]))),
                                     order_key(__float_as_uint(fmaxf(high[2], high[3])))};
            return bound_value(reached_by<T>(key, p.top));
          }
          uint32_t key[U];
#pragma unroll
          for (int q = 0; q < U; ++q) key[q] = order_key(__float_as_uint(high[q]));
          return bound_value(reached_by<T>(key, p.top));
        };
        bool fresh = batch == 0;               // K of the batch's own elements reach the limit
        if (fresh) limit = reach();
        if (__ballot(top >= limit)) {
          // The thread's elements from `from` on, a bit each.
          auto reaching = [&](float from) __attribute__((always_inline)) {
            hold(cur);
            uint32_t pass = 0;
#pragma unroll
            for (int q = U - 1; q >= 0; --q) {
              float v[V];
              IO::unpack(cur[q], v);
#pragma unroll
              for (int e = V - 1; e >= 0; --e) pass = pass + pass + (v[e] >= from ? 1u : 0u);
            }
            return pass;
          };
          auto all = [&](uint32_t n) __attribute__((always_inline)) {
            return __builtin_amdgcn_readlane((int)wave_upto(n), 63);
          };
          uint32_t pass = reaching(limit);
          if (limit == -INFINITY)              // which is also what lies outside the row
#pragma unroll
            for (int q = 0; q < U; ++q)
#pragma unroll
              for (int e = 0; e < V; ++e)
                if (!has(c + q * NT, e)) pass &= ~(1u << (V * q + e));
          // More than a batch in no order has, or than the list holds: a rising row, runs of
          // equal values. (Thirty-two elements to a lane: few lanes cannot.)
          const int most = min(2 * p.top + 32, kCap - listed);
          if (__builtin_expect(32 * __popcll(__ballot(pass != 0)) > most && all(__popc(pass)) > most, 0)) {
            const float to = fresh ? limit : reach();
            if (to >= limit) {                 // K of this batch make it the limit
              fresh = true;
              limit = to;
              keep(sh.list, listed, order_key(__float_as_uint(to)));
              pass &= reaching(to);
              // Those above it, and of those at it the first few that make K.
              const uint32_t strict = pass & reaching(above(to));
              const int want = max(0, p.top - all(__popc(strict)));
              int before = 0;
#pragma unroll 1
              for (int q = 0; q < U; ++q) {
                uint32_t f = (pass & ~strict) >> (V * q) & ((1u << V) - 1);
                const int n = __popc(f), upto = (int)wave_upto((uint32_t)n);
                const int stay = min(max(want - before - (upto - n), 0), n);
#pragma unroll 1
                for (int x = n; x > stay; --x) {
                  const uint32_t last = 0x80000000u >> __clz(f);
                  f ^= last;
                  pass ^= last << (V * q);
                }
                before += __builtin_amdgcn_readlane(upto, 63);
              }
            }
          }
          for (uint64_t any; (any = __ballot(pass != 0));) {
            const uint32_t i = pass ? __ffs(pass) - 1 : 0;
            const int at = listed + (int)__builtin_amdgcn_mbcnt_hi((uint32_t)(any >> 32),
                                                                   __builtin_amdgcn_mbcnt_lo((uint32_t)any, 0));
            uint32_t w = cur[0][0];
#pragma unroll
            for (uint32_t u = 1; u < 4 * U; ++u) w = i / (V / 4) == u ? cur[u / 4][u % 4] : w;
            float v[V];
            IO::unpack(u32x4{w, w, w, w}, v);
            const float x1 = V == 8 && (i & 1) ? v[1] : v[0];
            if (pass && at < kCap) sh.list[at] = rank_key(x1, rc.first(c + (int)(i / V) * NT) + (int)(i % V));
            pass &= pass - 1;
            listed += __popcll(any);
          }
        }
        over |= listed > kCap;
        listed = min(listed, kCap);
        if (fresh) limit = above(limit);       // an equal value at a higher place ranks lower
        // after batches 1, 3, 7, ...; of many alternatives after the first as well
        if (more && ((((batch + 1) & batch) == 0 && (batch || p.top > 16)) || listed > kCap / 2) && listed >= p.top) {
          limit = fmaxf(limit, above(bound_value(refine_list<T>(sh.list, listed, p.top))));
        }
      }
      if (!more) break;
    }

    // The sums relative to the maximum.
    Sums v;
    v.m = m;
    {
      const float off = fmaf(-m, kLog2e, r);
      const float f = __builtin_amdgcn_exp2f(off);
      v.s = s * f;
      v.t = kLn2 * f * fmaf(s, off, t);
      if (m == -INFINITY) v = {kLowest, s, 0.0f};                    // s: 0, or NaN
    }
    v = moved(v, wave_max(v.m));
    v.s = wave_sum(v.s);
    v.t = wave_sum(v.t);
    // NaN and +inf (S is not finite then), or a maximum of over 64. (S may be 0 there: r does
    // not move for elements below -992 / log2 e, whose 2^(x log2 e - r) may all be too small.)
    const bool some = __ballot(m != -INFINITY);
    const bool odd = !(v.s < INFINITY) || (some && !(fabsf(v.m) <= 64.0f));
    if (odd) {
      float s2 = 0.0f, t2 = 0.0f;
      for (int c = c0 + tid; c < c1 && rc.any(c); c += NT) {
        float y[V];
        IO::unpack(rc.load(x, c, none), y);
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const float d = y[e] - v.m, w = __builtin_amdgcn_exp2f(d * kLog2e);
          s2 += w;
          t2 += w == 0.0f ? 0.0f : w * d;
        }
      }
      v.s = wave_sum(s2);
      v.t = wave_sum(t2);
    }
    if (some && v.s < 1.0f) v.s = 1.0f;        // (NaN stays)
    if (v.t > 0.0f) v.t = 0.0f;
    int found = 0;
    if constexpr (TOP) {
      if (!over && v.s < INFINITY) {
        found = finish<T>(sh, p.top, listed);
      } else {                                 // the largest below the last one, K times
        uint64_t last = ~0ull;
        for (int i = 0; i < p.top; ++i) {
          uint64_t best = 0;
          for (int c = c0 + tid; c < c1 && rc.any(c); c += NT) {
            float y[V];
            IO::unpack(rc.load(x, c, none), y);
#pragma unroll
            for (int e = 0; e < V; ++e) {
              const uint64_t k = rank_key(y[e], rc.first(c) + e);
              // (NaN at place 0 is the largest key of all)
              if (rc.has(c, e) && (i == 0 || k < last) && k > best) best = k;
            }
          }
#pragma unroll
          for (int o = 32; o; o >>= 1) best = max(best, (uint64_t)__shfl_xor((unsigned long long)best, o));
          last = best;
          if (tid == 0) sh.best[i] = last;
        }
        found = p.top;
        __builtin_amdgcn_wave_barrier();
      }
    }
    if (p.pieces > 1) {
      if (tid == 0) {
        float* to = p.sums + job * 4;
        to[0] = v.m;
        to[1] = v.s;
        to[2] = v.t;
      }
      // (a piece of fewer elements: keys of none)
      if constexpr (TOP) {
        for (int i = tid; i < p.top; i += NT) p.keys[job * p.top + i] = i < found ? sh.best[i] : 0;
      }
    } else {
      const float ls = logf(v.s);
      if (tid == 0) {
        p.lse[row] = v.m + ls;
        if (p.entropy) p.entropy[row] = ls - v.t / v.s;
        if (p.tokens) {
          const int k = p.tokens[row];
          p.logprob[row] = (uint32_t)k < (uint32_t)p.vocab ? (IO::ld(x, k) - v.m) - ls : 0.0f;
        }
      }
      if constexpr (TOP)
        for (int i = tid; i < p.top; i += NT) {
          const uint64_t k = sh.best[i];
          p.top_index[row * p.top + i] = key_place(k);
          p.top_logprob[row * p.top + i] = (key_value(k) - v.m) - ls;
        }
    }
    __builtin_amdgcn_wave_barrier();           // the next row's list
  }
}

// A row's pieces: the sums of all, and the largest of their keys.
template <NormType T>
__global__ __launch_bounds__(256) void logprob_join(LParams p) {
  using IO = Io<T>;
  __shared__ __attribute__((aligned(16))) uint64_t list[kMaxKeys], some[2 * kMaxTop + kMaxPieces];
  __shared__ uint64_t threshold;
  __shared__ int count;
  const int tid = threadIdx.x, lane = tid & 63;
  for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
    const uint8_t* x = p.x + row * p.x_rs * (int64_t)(16 / IO::kVec);
    const float* from = p.sums + row * p.pieces * 4;
    Sums v = {kLowest, 0.0f, 0.0f};
    if (lane < p.pieces) v = {from[4 * lane], from[4 * lane + 1], from[4 * lane + 2]};
    const uint64_t* keys = p.keys + row * p.pieces * p.top;
    const int n = p.pieces * p.top;
    for (int i = tid; i < n; i += 256) list[i] = keys[i];
    v = moved(v, wave_max(v.m));
    v.s = wave_sum(v.s);
    v.t = wave_sum(v.t);
    const float ls = logf(v.s);
    if (tid == 0) {
      p.lse[row] = v.m + ls;
      if (p.entropy) p.entropy[row] = ls - v.t / v.s;
      if (p.tokens) {
        const int k = p.tokens[row];
        p.logprob[row] = (uint32_t)k < (uint32_t)p.vocab ? (IO::ld(x, k) - v.m) - ls : 0.0f;
      }
    }
    if (!p.top) continue;
    // K keys reach the K-th largest of the pieces' first ceil(K / pieces) ones: only
    // what reaches it as well is ranked.
    const int first = (p.top + p.pieces - 1) / p.pieces, m = first * p.pieces;
    if (tid == 0) {
      threshold = 0;
      count = 0;
    }
    __syncthreads();
    if (tid < m) some[tid] = list[tid / first * p.top + tid % first];
    __syncthreads();
    if (tid < m && some[tid] && rank_of(some, m, some[tid]) == p.top - 1) threshold = some[tid];
    __syncthreads();
    const uint64_t bound = max((uint64_t)1, threshold);
    uint64_t mine[kMaxKeys / 256];
#pragma unroll
    for (int q = 0; q < kMaxKeys / 256; ++q) mine[q] = tid + 256 * q < n ? list[tid + 256 * q] : 0;
    __syncthreads();
#pragma unroll
    for (int q = 0; q < kMaxKeys / 256; ++q)
      if (mine[q] >= bound) list[atomicAdd(&count, 1)] = mine[q];
    __syncthreads();
    const int c = count;
    for (int i = tid; i < c; i += 256) {
      const uint64_t k = list[i];
      const int at = rank_of(list, c, k);
      if (at < p.top) {
        p.top_index[row * p.top + at] = key_place(k);
        p.top_logprob[row * p.top + at] = (key_value(k) - v.m) - ls;
      }
    }
    __syncthreads();
  }
}

// ---- backward ------------------------------------------------------------------

struct GParams {
  const uint8_t* x;
  uint8_t* dx;
  int64_t x_rs, dx_rs, rows;
  int vocab;
  const int* tokens;
  const float* lse; const float* entropy;
  const float* dlogprob; const float* dentropy;
};

// kU chunks of a row per thread: blockIdx.x along the row, blockIdx.y over the rows.
template <NormType T, bool AL, bool ENT>
__global__ __launch_bounds__(256) void logprob_grad(GParams p) {
  using IO = Io<T>;
  constexpr int V = IO::kVec;
  for (int64_t row = blockIdx.y; row < p.rows; row += gridDim.y) {
    const uint8_t* x = p.x + row * p.x_rs * (int64_t)(16 / V);
    uint8_t* dx = p.dx + row * p.dx_rs * (int64_t)(16 / V);
    const float lse = p.lse[row];
    const int token = p.tokens ? p.tokens[row] : -1;
    const bool given = (uint32_t)token < (uint32_t)p.vocab;
    const float g = given ? p.dlogprob[row] : 0.0f;
    const float gh = ENT ? p.dentropy[row] : 0.0f;
    const float c0 = ENT ? fmaf(gh, p.entropy[row], g) : g;
    const bool some = given || gh != 0.0f;   // else the row has no gradient, whatever is in it
    const RowChunks<T, AL> rc(x, p.vocab, V - 1);
    const int first = blockIdx.x * 256 * kU + threadIdx.x;
    u32x4 raw[kU];
#pragma unroll
    for (int q = 0; q < kU; ++q)
      if (rc.any(first + 256 * q)) raw[q] = rc.load(x, first + 256 * q, u32x4{0, 0, 0, 0});
#pragma unroll
    for (int q = 0; q < kU; ++q) {
      const int c = first + 256 * q;
      if (!rc.any(c)) continue;
      float v[V];
      IO::unpack(raw[q], v);
#pragma unroll
      for (int e = 0; e < V; ++e) {
        float lp = v[e] - lse;
        // where p is 0 the entropy term is, whatever log p is (NaN stays)
        if constexpr (ENT) lp = lp < -200.0f ? -200.0f : lp;
        const float w = __builtin_amdgcn_exp2f(lp * kLog2e);
        const float a = ENT ? fmaf(gh, lp, c0) : c0;
        v[e] = some ? -(w * a) : 0.0f;
      }
      const uint32_t at = (uint32_t)token - (uint32_t)rc.first(c);
      if (given && at < (uint32_t)V) {
#pragma unroll
        for (int e = 0; e < V; ++e)
          if ((uint32_t)e == at) v[e] += g;
      }
      rc.store(dx, c, IO::pack(v));
    }
  }
}

// ---- launch ----------------------------------------------------------------------

bool on16(const void* q) { return (uintptr_t)q % 16 == 0; }

struct Plan {
  int pieces, each;
  size_t sums, keys;     // bytes of the workspace
};

// A wave to a row, or to each of a row's pieces where rows are fewer than two waves to a
// SIMD: of at least a batch, and not more than the join holds. us for 1, 2 and 4 waves to
// a SIMD at least: 256 x 131072 bf16, 8 alternatives, - / 28.9 / 30.9; 2048 x 32000
// without any 24.9 in one piece, 32.8 in four. Four waves to a row, a workgroup with
// barriers: 40 us for 19 at 8192 x 4000, 84 for 86 at 4096 x 32001 fp32.
Plan plan_of(NormType t, int64_t rows, int vocab, int top) {
  Plan x{};
  const int V = t == NormType::F32 ? 4 : 8;
  const int chunks = (vocab + V - 1) / V + 1;        // one more where rows are off 16 bytes
  const int most = (chunks + kU * 64 - 1) / (kU * 64);
  x.pieces = (int)std::min<int64_t>({(2048 + rows - 1) / rows, most, kMaxPieces, kMaxKeys / std::max(1, top)});
  x.each = (chunks + x.pieces - 1) / x.pieces;
  if (x.pieces > 1) {
    x.sums = (size_t)rows * x.pieces * 16;
    x.keys = (size_t)rows * x.pieces * top * 8;
  }
  return x;
}

template <NormType T, bool AL>
hipError_t run_forward(const TokenLogProbDesc& d, const Plan& x, hipStream_t s) {
  LParams p{};
  p.x = (const uint8_t*)d.x; p.x_rs = d.x_row_stride; p.rows = d.rows; p.vocab = d.vocab; p.top = d.top;
  p.align_mask = Io<T>::kVec - 1;
  p.pieces = x.pieces; p.each = x.each;
  p.tokens = d.tokens; p.logprob = d.logprob; p.lse = d.lse; p.entropy = d.entropy;
  p.top_logprob = d.top_logprob; p.top_index = d.top_index;
  p.sums = (float*)d.ws;
  p.keys = (uint64_t*)((uint8_t*)d.ws + x.sums);
  const unsigned grid = (unsigned)std::min<int64_t>(d.rows * x.pieces, max_workgroups(64));
  if (d.top) hipLaunchKernelGGL((logprob_pieces<T, AL, true>), dim3(grid), dim3(64), 0, s, p);
  else hipLaunchKernelGGL((logprob_pieces<T, AL, false>), dim3(grid), dim3(64), 0, s, p);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess || x.pieces == 1) return e;
  hipLaunchKernelGGL(logprob_join<T>, dim3((unsigned)std::min<int64_t>(d.rows, max_workgroups(256))), dim3(256), 0, s, p);
  return hipGetLastError();
}

template <NormType T>
hipError_t run_forward(const TokenLogProbDesc& d, hipStream_t s) {
  const Plan x = plan_of(T, d.rows, d.vocab, d.top);
  const bool al = on16(d.x) && d.vocab % Io<T>::kVec == 0 && d.x_row_stride % Io<T>::kVec == 0;
  return al ? run_forward<T, true>(d, x, s) : run_forward<T, false>(d, x, s);
}

template <NormType T>
hipError_t run_grad(const TokenLogProbGradDesc& d, hipStream_t s) {
  constexpr int V = Io<T>::kVec;
  GParams p{};
  p.x = (const uint8_t*)d.x; p.dx = (uint8_t*)d.dx; p.x_rs = d.x_row_stride; p.dx_rs = d.dx_row_stride;
  p.rows = d.rows; p.vocab = d.vocab; p.tokens = d.tokens; p.lse = d.lse; p.entropy = d.entropy;
  p.dlogprob = d.dlogprob; p.dentropy = d.dentropy;
  const bool al = on16(d.x) && on16(d.dx) && d.vocab % V == 0 && d.x_row_stride % V == 0 && d.dx_row_stride % V == 0;
  const int chunks = (d.vocab + V - 1) / V + (al ? 0 : 1);
  const dim3 grid((unsigned)((chunks + 256 * kU - 1) / (256 * kU)), (unsigned)std::min<int64_t>(d.rows, 65535));
  auto go = [&](auto kern) { hipLaunchKernelGGL(kern, grid, dim3(256), 0, s, p); };
  if (al && d.entropy) go(logprob_grad<T, true, true>);
  else if (al) go(logprob_grad<T, true, false>);
  else if (d.entropy) go(logprob_grad<T, false, true>);
  else go(logprob_grad<T, false, false>);
  return hipGetLastError();
}

}  // namespace

size_t token_logprob_workspace(NormType t, int64_t rows, int vocab, int top) {
  const Plan x = plan_of(t, rows, vocab, top);
  return x.sums + x.keys;
}

hipError_t launch_token_logprob(NormType t, const TokenLogProbDesc& d, hipStream_t s) {
  switch (t) {
    case NormType::BF16: return run_forward<NormType::BF16>(d, s);
    case NormType::F16:  return run_forward<NormType::F16>(d, s);
    case NormType::F32:  return run_forward<NormType::F32>(d, s);
  }
  return hipErrorNotSupported;
}

hipError_t launch_token_logprob_grad(NormType t, const TokenLogProbGradDesc& d, hipStream_t s) {
  switch (t) {
    case NormType::BF16: return run_grad<NormType::BF16>(d, s);
    case NormType::F16:  return run_grad<NormType::F16>(d, s);
    case NormType::F32:  return run_grad<NormType::F32>(d, s);
  }
  return hipErrorNotSupported;
}

}  // namespace grxk
