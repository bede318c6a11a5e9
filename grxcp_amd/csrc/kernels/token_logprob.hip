// grxDNN log probabilities of given tokens over rows of logits, with entropy and
// the top alternatives, and their gradient in the logits, on gfx950.
//
// New: the reference plans softmax for grxDNN (ref
// docs/designs/grxcp_roadmap.md:864-877) and ships no code.
//
// Forward: one pass over the logits. A row, or a piece of it where rows are few,
// goes to a workgroup; every thread keeps
//   s = sum 2^(x log2 e - r),  t = sum 2^(x log2 e - r) (x log2 e - r)
// over its elements with a reference r of its own that moves only when a batch's
// maximum exceeds it by more than 8, so an element costs an unpack, half a max, two
// fmas, an add and an exp2: the exp2 (a quarter rate instruction) makes that 8.5
// lane operations against the 64 a CU does in a cycle, which is 8 TB/s of bf16, little
// above what the memory gives. Then log sum exp = max + log S and entropy =
// log S - T / S from the sums moved to the row's maximum.
// Products x log2 e are good to 2^-25 |x| (fma), which is enough within |x| <= 64:
// a row whose maximum is outside, or whose sums are not finite, is read again with
// x - max formed first (careful_sums).
//
// Alternatives: the same pass compares each batch's maximum with a threshold that K
// elements already read reach, and only where it is higher looks at the elements: those
// above go to a list in LDS. The first threshold is the K-th largest of the threads' (or
// groups of four threads') maxima over the first batch; it is raised after batches 4,
// 16, 64, ... from the list, so a row of random order pushes about K + 3 K + 3 K + ... of
// its elements. Elements are ranked by value, then by lower index; as batches come in
// index order an equal value later never outranks one in the list. A list that runs over (an
// ordered row), NaN and +inf take the direct way: the largest element below the last one,
// K times.
//
// Backward: one element-wise pass, bound by reading x and writing dx.

#include "../launch.h"
#include "device_common.h"
#include "paged_common.h"
#include "row_io.h"

#include <algorithm>

namespace grxk {
namespace {

constexpr float kLog2e = 1.4426950408889634f, kLog2eLow = 1.925963033e-8f, kLn2 = 0.6931471805599453f;
constexpr float kLowest = -__FLT_MAX__;
constexpr int kU = 4;         // chunks of a thread's batch
constexpr int kMaxTop = 64;
constexpr int kMaxPieces = 32;

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
__device__ __forceinline__ Sums both(Sums a, Sums b) {
  const float m = fmaxf(a.m, b.m);
  const float fa = __builtin_amdgcn_exp2f((a.m - m) * kLog2e), fb = __builtin_amdgcn_exp2f((b.m - m) * kLog2e);
  Sums r;
  r.m = m;
  r.s = fmaf(fa, a.s, fb * b.s);
  // the weight of a part of no sum is 0 however far its maximum is
  r.t = fa * a.t + fb * b.t;
  r.t += a.s != 0.0f && fa != 0.0f ? fa * a.s * (a.m - m) : 0.0f;
  r.t += b.s != 0.0f && fb != 0.0f ? fb * b.s * (b.m - m) : 0.0f;
  return r;
}
__device__ __forceinline__ Sums wave_both(Sums v) {
#pragma unroll
  for (int o = 32; o; o >>= 1) v = both(v, {__shfl_xor(v.m, o), __shfl_xor(v.s, o), __shfl_xor(v.t, o)});
  return v;
}

// Number of the c keys that are larger than k.
__device__ __forceinline__ int rank_of(const uint64_t* keys, int c, uint64_t k) {
  int r = 0;
#pragma unroll 4
  for (int i = 0; i < c; ++i) r += keys[i] > k;
  return r;
}

template <int NW> __device__ __forceinline__ void sync() {
  if constexpr (NW > 1) __syncthreads();
  else __builtin_amdgcn_wave_barrier();
}

template <int NW>
struct Shared {
  static constexpr int kCap = NW == 1 ? 512 : 1024;   // keys of the list
  Sums sums[NW];
  uint64_t list[kCap], best[kMaxTop];
  uint64_t groups[64 * NW];
  uint64_t threshold;
  int count;
};

// The list's K largest keys in order at its front, and the K-th as the threshold.
template <int NW>
__device__ __forceinline__ void shorten(Shared<NW>& sh, int top) {
  const int tid = threadIdx.x;
  sync<NW>();
  const int c = min(sh.count, Shared<NW>::kCap);
  for (int i = tid; i < c; i += 64 * NW) {
    const uint64_t k = sh.list[i];
    const int r = rank_of(sh.list, c, k);
    if (r < top) sh.best[r] = k;
  }
  sync<NW>();
  if (tid < min(c, top)) sh.list[tid] = sh.best[tid];
  if (tid == 0 && c >= top) {
    sh.threshold = sh.best[top - 1];
    sh.count = top;
  }
  sync<NW>();
}

// One piece of a row per workgroup of NW waves.
template <NormType T, bool AL, int NW, bool TOP>
__global__ __launch_bounds__(64 * NW) void logprob_pieces(LParams p) {
  using IO = Io<T>;
  constexpr int V = IO::kVec, NT = 64 * NW;
  constexpr uint32_t kNone = T == NormType::F32 ? 0xff800000u : T == NormType::BF16 ? 0xff80ff80u : 0xfc00fc00u;
  const u32x4 none = {kNone, kNone, kNone, kNone};     // -inf: outside the row
  __shared__ Shared<NW> sh;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t jobs = p.rows * p.pieces;
  for (int64_t job = blockIdx.x; job < jobs; job += gridDim.x) {
    const int64_t row = p.pieces == 1 ? job : job / p.pieces;
    const int piece = p.pieces == 1 ? 0 : (int)(job - row * p.pieces);
    const uint8_t* x = p.x + row * p.x_rs * (int64_t)(16 / V);
    const RowChunks<T, AL> rc(x, p.vocab, p.align_mask);
    const int c0 = piece * p.each, c1 = p.pieces == 1 ? INT_MAX : c0 + p.each;
    auto load = [&](int c) __attribute__((always_inline)) { return c < c1 && rc.any(c) ? rc.load(x, c, none) : none; };
    // Places of chunk c that are in the row and the piece.
    auto has = [&](int c, int e) __attribute__((always_inline)) { return c < c1 && rc.any(c) && rc.has(c, e); };

    // Only the packed batch stays in registers between the passes over it.
    auto hold = [&](u32x4 (&w)[kU]) __attribute__((always_inline)) {
#pragma unroll
      for (int q = 0; q < kU; ++q) asm volatile("" : "+v"(w[q]));
    };
    if (tid == 0) sh.count = 0;
    float m = -INFINITY, r = -1000.0f, s = 0.0f, t = 0.0f;
    float limit = -INFINITY;                   // values above it may be alternatives
    bool over = false;                         // the list lost some
    u32x4 raw[kU];
#pragma unroll
    for (int q = 0; q < kU; ++q) raw[q] = load(c0 + tid + NT * q);
    for (int c = c0 + tid, batch = 0;; c += kU * NT, ++batch) {
      u32x4 cur[kU];
#pragma unroll
      for (int q = 0; q < kU; ++q) cur[q] = raw[q];
      // (uniform: the first thread's next chunk)
      const int next = c - tid + kU * NT;
      const bool more = next < c1 && rc.any(next);
      if (more)
#pragma unroll
        for (int q = 0; q < kU; ++q) raw[q] = load(c + (kU + q) * NT);
      float high[kU];
#pragma unroll
      for (int q = 0; q < kU; ++q) {
        float v[V];
        IO::unpack(cur[q], v);
        high[q] = v[0];
#pragma unroll
        for (int e = 1; e < V; ++e) high[q] = fmaxf(high[q], v[e]);
      }
      const float top = fmaxf(fmaxf(high[0], high[1]), fmaxf(high[2], high[3]));
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
      for (int q = 0; q < kU; ++q) {
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
#pragma unroll
        for (int q = 0; q < kU; ++q) {
          float v[V];
          IO::unpack(cur[q], v);
#pragma unroll
          for (int e = 0; e < V; ++e) {
            const float d = fmaf(v[e], kLog2e, -r), w = __builtin_amdgcn_exp2f(d);
            bt += w == 0.0f ? 0.0f : w * d;
          }
        }
      }
      s += bs;
      t += bt;
      if constexpr (TOP) {
        hold(cur);
        uint64_t bound = 0;                    // first batch: keys from here on
        if (batch == 0) {
          // The K-th largest of the threads' own largest keys, or of groups of four
          // threads' where K is small; fewer than K such keys: every element is listed.
          uint64_t best = 0;
#pragma unroll
          for (int q = kU - 1; q >= 0; --q) {
            float v[V];
            IO::unpack(cur[q], v);
            const int at = c + q * NT;
#pragma unroll
            for (int e = V - 1; e >= 0; --e)
              if (has(at, e)) best = max(best, rank_key(v[e], rc.first(at) + e));
          }
          const bool by4 = NW > 1 && p.top <= 16;
          if (by4) {
            best = max(best, (uint64_t)__shfl_xor((unsigned long long)best, 1));
            best = max(best, (uint64_t)__shfl_xor((unsigned long long)best, 2));
            if ((tid & 3) == 0) sh.groups[tid >> 2] = best;
          } else {
            sh.groups[tid] = best;
          }
          if (tid == 0) sh.threshold = 0;
          sync<NW>();
          const int n = by4 ? NT / 4 : NT;
          if (tid < n) {
            const uint64_t k = sh.groups[tid];
            if (k && rank_of(sh.groups, n, k) == p.top - 1) sh.threshold = k;
          }
          sync<NW>();
          bound = sh.threshold;
          hold(cur);
        }
#pragma unroll
        for (int q = 0; q < kU; ++q) {
          if (batch && !__ballot(high[q] > limit)) continue;
          float v[V];
          IO::unpack(cur[q], v);
          const int at = c + q * NT;
#pragma unroll
          for (int e = 0; e < V; ++e) {
            const bool in = batch ? v[e] > limit : has(at, e) && rank_key(v[e], rc.first(at) + e) >= bound;
            if (in) {
              const int to = atomicAdd(&sh.count, 1);
              if (to < sh.kCap) sh.list[to] = rank_key(v[e], rc.first(at) + e);
            }
          }
        }
        if (batch == 0) limit = bound ? key_value(bound) : -INFINITY;
        // after batches 0, 3, 15, 63, ... (the list's order does not depend on the waves')
        if (more && ((batch + 1) & batch) == 0 && (__ffs(batch + 1) & 1)) {
          sync<NW>();
          over |= sh.count > sh.kCap;
          shorten<NW>(sh, p.top);
          limit = key_value(sh.threshold);
        }
      }
      if (!more) break;
    }

    // The sums relative to the maximum.
    Sums v;
    v.m = m;
    {
      const float off = fmaf(-m, kLog2eLow, fmaf(-m, kLog2e, r));    // r - m log2 e
      const float f = __builtin_amdgcn_exp2f(off);
      v.s = s * f;
      v.t = kLn2 * f * fmaf(s, off, t);
      if (m == -INFINITY) v = {kLowest, s, 0.0f};                    // s: 0, or NaN
    }
    v = wave_both(v);
    if (lane == 0) sh.sums[wave] = v;
    sync<NW>();
    v = sh.sums[0];
#pragma unroll
    for (int w = 1; w < NW; ++w) v = both(v, sh.sums[w]);
    // NaN and +inf (S is not finite then), or a maximum of over 64.
    const bool odd = !(v.s < INFINITY) || (!(fabsf(v.m) <= 64.0f) && v.s != 0.0f);
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
      const float sum = wave_sum(s2), tsum = wave_sum(t2);
      sync<NW>();
      if (lane == 0) sh.sums[wave] = {v.m, sum, tsum};
      sync<NW>();
      v.s = v.t = 0.0f;
#pragma unroll
      for (int w = 0; w < NW; ++w) {
        v.s += sh.sums[w].s;
        v.t += sh.sums[w].t;
      }
    }
    if constexpr (TOP) {
      over |= sh.count > sh.kCap;
      if (!over && v.s < INFINITY) {
        shorten<NW>(sh, p.top);
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
              if (rc.has(c, e) && k < last && k > best) best = k;
            }
          }
#pragma unroll
          for (int o = 32; o; o >>= 1) best = max(best, (uint64_t)__shfl_xor((unsigned long long)best, o));
          sync<NW>();
          if (lane == 0) sh.groups[wave] = best;
          sync<NW>();
          last = sh.groups[0];
#pragma unroll
          for (int w = 1; w < NW; ++w) last = max(last, sh.groups[w]);
          if (tid == 0) sh.list[i] = last;
        }
        sync<NW>();
        if (tid == 0) sh.count = p.top;
        sync<NW>();
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
        const int n = min(sh.count, p.top);
        for (int i = tid; i < p.top; i += NT) p.keys[job * p.top + i] = i < n ? sh.list[i] : 0;
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
          const uint64_t k = sh.list[i];
          p.top_index[row * p.top + i] = key_place(k);
          p.top_logprob[row * p.top + i] = (key_value(k) - v.m) - ls;
        }
    }
    sync<NW>();                                // the next row's list
  }
}

// A row's pieces: the sums of all, and the largest of their keys.
template <NormType T>
__global__ __launch_bounds__(256) void logprob_join(LParams p) {
  using IO = Io<T>;
  __shared__ uint64_t list[kMaxPieces * kMaxTop], some[2 * kMaxTop + kMaxPieces];
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
    v = wave_both(v);
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
    uint64_t mine[kMaxPieces * kMaxTop / 256];
#pragma unroll
    for (int q = 0; q < kMaxPieces * kMaxTop / 256; ++q) mine[q] = tid + 256 * q < n ? list[tid + 256 * q] : 0;
    __syncthreads();
#pragma unroll
    for (int q = 0; q < kMaxPieces * kMaxTop / 256; ++q)
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
        // without a token and an entropy the row has no gradient, whatever is in it
        v[e] = ENT || given ? -(w * a) : 0.0f;
      }
      const int at = token - rc.first(c);
      if (given && (uint32_t)at < (uint32_t)V) {
#pragma unroll
        for (int e = 0; e < V; ++e)
          if (e == at) v[e] += g;
      }
      rc.store(dx, c, IO::pack(v));
    }
  }
}

// ---- launch ----------------------------------------------------------------------

bool on16(const void* q) { return (uintptr_t)q % 16 == 0; }

struct Plan {
  int nw, pieces, each;
  size_t sums, keys;     // bytes of the workspace
};

Plan plan_of(NormType t, int64_t rows, int vocab, int top) {
  Plan x{};
  const int V = t == NormType::F32 ? 4 : 8;
  const int chunks = (vocab + V - 1) / V + 1;        // one more where rows are off 16 bytes
  x.nw = chunks <= kU * 64 ? 1 : 4;
  // Few rows: pieces of at least a batch, four workgroups to a CU.
  const int batch = kU * 64 * x.nw, most = (chunks + batch - 1) / batch;
  x.pieces = (int)std::max<int64_t>(1, std::min<int64_t>({(1024 + rows - 1) / rows, most, kMaxPieces}));
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
  const unsigned grid = (unsigned)std::min<int64_t>(d.rows * x.pieces, max_workgroups(64 * x.nw));
  auto go = [&](auto kern) { hipLaunchKernelGGL(kern, dim3(grid), dim3(64 * x.nw), 0, s, p); };
  if (x.nw == 1 && d.top) go(logprob_pieces<T, AL, 1, true>);
  else if (x.nw == 1) go(logprob_pieces<T, AL, 1, false>);
  else if (d.top) go(logprob_pieces<T, AL, 4, true>);
  else go(logprob_pieces<T, AL, 4, false>);
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
