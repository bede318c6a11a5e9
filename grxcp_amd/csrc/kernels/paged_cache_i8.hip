// grxDNN paged key-value cache in 8 bits on gfx950: rows quantised as they are written,
// and read back.
//
// New: the reference plans attention for grxDNN (ref
// docs/designs/grxcp_roadmap.md:864-877) and ships neither it nor a cache.
//
// A block of `block` slots of one head has one scale, the largest magnitude / 127
// rounded up to 8 significant bits. With that a quotient x / scale of a 16-bit value is
// either half way between two codes or further from there than 2^-17 of it: |x / s - (k + 1/2)|
// = |2x - (2k + 1) s| / 2s is a whole number of the smaller last bit of 2x and s, and that
// is at least 1 / 2S (S < 2^8 the significand of s) or 1 / X of the quotient (X < 2^11 that
// of x; 2^15 for a code times an older scale). So codes are the same in every arithmetic
// that keeps 2^-17 and tells a tie.

#include "../launch.h"
#include "device_common.h"
#include "paged_common.h"
#include "row_io.h"

#include <algorithm>

namespace grxk {
namespace {

constexpr int kThreads = 256;
constexpr int64_t kStream = 32 << 20;     // bytes of 16 bits from which on stores go past the caches

// A pool of codes as the kernels address it, strides in bytes, and its scales.
struct Pool8 {
  uint8_t* p;
  int64_t sp, sh, ss;
  float* scale;
  int64_t cp, ch, cb;
  __device__ __forceinline__ uint8_t* row(int page, int h, int slot) const {
    return p + page * sp + h * sh + slot * ss;
  }
  __device__ __forceinline__ float* scale_of(int page, int h, int block) const {
    return scale + page * cp + h * ch + block * cb;
  }
};
Pool8 pool_of(const PagedCache& c, const QuantScales& q, bool values) {
  return values ? Pool8{(uint8_t*)c.v, c.v_sp, c.v_sh, c.v_ss, q.v, q.sp, q.sh, q.sb}
                : Pool8{(uint8_t*)c.k, c.k_sp, c.k_sh, c.k_ss, q.k, q.sp, q.sh, q.sb};
}
PagedView view_of(const PagedCache& c) {
  return {c.table, c.table_rs, c.lengths, c.pages, c.page, c.W * c.page, page_div(c.page)};
}

// ---- append ------------------------------------------------------------------

struct NewRows {
  const uint8_t* p;
  int64_t sb, sh, st;    // bytes
};
struct AppendParams {
  PagedView view;
  Pool8 pool[2];
  NewRows rows[2];
  const int* counts;
  PageDiv by_heads, by_block;
  int B, T, heads, block;
};

template <NormType T> __device__ __forceinline__ float half_value(uint32_t bits) {
  return T == NormType::BF16 ? bf16_to_f32((uint16_t)bits) : f16_to_f32((uint16_t)bits);
}

// The scale of values of which `bits` (of the 16-bit type, no sign) is the largest
// magnitude: NaN if that is an infinity or NaN.
template <NormType T> __device__ __forceinline__ float scale_for(uint32_t bits) {
  const float most = half_value<T>(bits);
  if (!(most <= __FLT_MAX__)) return __uint_as_float(0x7fc00000u);
  if (most == 0.0f) return 0.0f;
  const uint32_t up = (__float_as_uint(most / 127.0f) + 0xffffu) & 0xffff0000u;
  return fmaxf(__uint_as_float(up), 0x1p-126f);
}

// 1 / s, less and more by 2^-21 of it: above what its rounding loses, far below the distance
// of a quotient from a half that it is not.
struct Inverse { float lo, hi; };
__device__ __forceinline__ Inverse inverse(float s) {
  const float r = 1.0f / s;
  return {r * (1.0f - 0x1p-21f), r * (1.0f + 0x1p-21f)};
}
// The codes of 4 values: x / s rounded to the nearest whole number, ties to the even one. 1.5 *
// 2^23 + x / s is rounded from either side of the quotient: to the same number, or, for a tie,
// to its two neighbours. Their sum has one bit fewer, so that it rounds to twice the even one,
// and the code is its low byte. (With the quotient's remainder, as a division corrects it,
// 23.9 for 23.2 us in the case below.)
__device__ __forceinline__ uint32_t codes4(const float* x, Inverse r) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    w[i] = __float_as_uint(fmaf(x[i], r.lo, 12582912.0f) + fmaf(x[i], r.hi, 12582912.0f));
  const uint32_t lo = __builtin_amdgcn_perm(w[1], w[0], 0x0c0c0400u);
  const uint32_t hi = __builtin_amdgcn_perm(w[3], w[2], 0x0c0c0400u);
  return lo | hi << 16;
}

// The same of scales of any bits, which only a caller sets: 64-bit quotients.
__device__ __forceinline__ bool few_bits(float s) { return (__float_as_uint(s) & 0xffffu) == 0; }
__device__ __forceinline__ u32x2 codes8(const float* x, double times, double s) {
  u32x2 w = {0, 0};
#pragma unroll
  for (int e = 0; e < 8; ++e) w[e / 4] |= ((uint32_t)(int)rint(x[e] * times / s) & 255u) << 8 * (e % 4);
  return w;
}

typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));

template <int CTRL> __device__ __forceinline__ uint32_t dpp_max(uint32_t v) {
  return max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, CTRL, 0xf, 0xf, false));
}
// The largest over L neighbouring lanes (4 to 64), in each.
template <int L> __device__ __forceinline__ uint32_t lanes_max(uint32_t v) {
  v = dpp_max<0xb1>(v);
  v = dpp_max<0x4e>(v);
  if constexpr (L >= 8) v = dpp_max<0x141>(v);
  if constexpr (L >= 16) v = dpp_max<0x140>(v);
  if constexpr (L >= 32) {
    const auto a = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    v = max(a[0], a[1]);
  }
  if constexpr (L == 64) {
    const auto b = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    v = max(b[0], b[1]);
  }
  return v;
}

// One task: the block of one head's keys or values (blockIdx.z) that gets new rows, by L
// threads with N chunks of 8 values each, held in registers between the maximum and the
// codes: read once. The threads take M tasks at a time. Rows that the block already holds are
// rounded again, to the new scale, where that is larger. us, 8 sequences of 500 to 4000 tokens
// of 8 heads of 128, blocks of 32: 22.4 (4.9 TB/s; stores through the caches 1.6 more,
// registers for eight waves a SIMD, which the loads then wait in turn for, 3.2), bound by memory
// with the VALU at work in 47 % of the cycles; one token of 64 sequences 5.5, a launch and the
// chain of length, table entry and rows. Where every block's scale grows rows are loaded,
// rounded and stored one after the other: one token of 64 sequences without / with, blocks of
// 16 4.7 / 4.9, of 64 5.6 / 6.1, of 256 8.9 / 12.3.
template <NormType T, int C, int L, int N, int M, bool STREAM>   // C: chunks of a row
__global__ __launch_bounds__(kThreads, 4) void append_i8(AppendParams p) {
  constexpr int P = kThreads / L;
  __shared__ uint32_t most_of[kThreads / 64];
  const int tid = threadIdx.x, l = tid % L;
  const Pool8& pool = p.pool[blockIdx.z];
  const NewRows& in = p.rows[blockIdx.z];
  for (int b = blockIdx.y; b < p.B; b += gridDim.y) {
    const int n = clamp_length(p.view.lengths[b], p.view.room);
    const int count = min(p.counts ? min(p.counts[b], p.T) : p.T, p.view.room - n);   // the others have no place
    if (count <= 0) continue;
    const int b0 = div_page(p.by_block, n), blocks = div_page(p.by_block, n + count - 1) - b0 + 1;
    const int64_t tasks = (int64_t)blocks * p.heads;
    for (int64_t t0 = (int64_t)blockIdx.x * (P * M); t0 < tasks; t0 += (int64_t)gridDim.x * (P * M)) {
      u32x4 x[M][N];
      int h[M], lo[M], page[M], row[M];                       // head, first slot, its place
      bool there[M];
      float before[M], now[M];
      int rest = 0;
#pragma unroll
      for (int m = 0; m < M; ++m) {
        const int64_t task = t0 + m * P + tid / L;
        const bool mine = task < tasks;
        const int at = mine ? (int)task : 0;
        const int j = div_page(p.by_heads, at);
        h[m] = at - j * p.heads;
        lo[m] = (b0 + j) * p.block;
        const int old = max(0, n - lo[m]), end = min(p.block, n + count - lo[m]);
        there[m] = find_slot(p.view, b, lo[m], &page[m], &row[m]) & mine;
        before[m] = there[m] && old > 0 ? *pool.scale_of(page[m], h[m], div_page(p.by_block, row[m])) : 0.0f;
        const uint8_t* src = in.p + b * in.sb + h[m] * in.sh;
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const int c = i * L + l, r = c / C;
          x[m][i] = u32x4{0, 0, 0, 0};
          if (there[m] && r >= old && r < end)
            x[m][i] = __builtin_nontemporal_load((const u32x4*)(src + (int64_t)(lo[m] + r - n) * in.st) + c % C);
        }
      }
#pragma unroll
      for (int m = 0; m < M; ++m) {
        const int old = max(0, n - lo[m]), end = min(p.block, n + count - lo[m]);
        u16x2 both = {0, 0};                                  // largest magnitudes of either half of a word
#pragma unroll
        for (int i = 0; i < N; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            both = __builtin_elementwise_max(both, __builtin_bit_cast(u16x2, x[m][i][e] & 0x7fff7fffu));
        uint32_t most = max(both[0], both[1]);
        if constexpr (L <= 64) {
          most = lanes_max<L>(most);
        } else {
          most = lanes_max<64>(most);
          __syncthreads();                                    // the task before has read
          if ((tid & 63) == 0) most_of[tid >> 6] = most;
          __syncthreads();
          most = max(max(most_of[0], most_of[1]), max(most_of[2], most_of[3]));
        }
        if (!there[m]) continue;                              // (L = 256: of the whole workgroup)
        const float need = scale_for<T>(most);
        float s = fmaxf(need, before[m]);
        if (s > 0.0f) s = fmaxf(s, 0x1p-126f);
        if (need != need || before[m] != before[m]) s = __uint_as_float(0x7fc00000u);
        const bool fine = s > 0.0f && s <= __FLT_MAX__;
        const Inverse inv = inverse(fine ? s : 1.0f);
        const bool grew = old > 0 && s > before[m] && fine;
        const bool many_bits = fine && !(few_bits(s) && (!grew || few_bits(before[m])));
        if (l == 0) *pool.scale_of(page[m], h[m], div_page(p.by_block, row[m])) = s;
        if (many_bits) {
          rest |= 1 << m;
          now[m] = s;
          continue;
        }
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const int c = i * L + l, r = c / C;
          if (r < old || r >= end) continue;
          float f[8];
          Io<T>::unpack(x[m][i], f);
          u32x2 w = {codes4(f, inv), codes4(f + 4, inv)};
          if (!fine) w = u32x2{0, 0};
          u32x2* to = (u32x2*)(pool.row(page[m], h[m], row[m] + r) + 8 * (c % C));
          if constexpr (STREAM) __builtin_nontemporal_store(w, to);
          else *to = w;
        }
        if (grew) {
          for (int i = 0; i < N; ++i) {
            const int c = i * L + l, r = c / C;
            if (r >= old) continue;
            u32x2* to = (u32x2*)(pool.row(page[m], h[m], row[m] + r) + 8 * (c % C));
            u32x2 w = *to;
            float f[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) f[e] = (float)(int8_t)(w[e / 4] >> 8 * (e % 4)) * before[m];
            *to = u32x2{codes4(f, inv), codes4(f + 4, inv)};
          }
        }
      }
      if (rest == 0) continue;
      // tasks with scales of many bits, apart from what the others hold in registers
#pragma unroll 1
      for (int m = 0; m < M; ++m) {
        if (!(rest >> m & 1)) continue;
        const float s = m ? now[M - 1] : now[0], was = m ? before[M - 1] : before[0];
        const int at = (int)(t0 + m * P + tid / L), j = div_page(p.by_heads, at), head = at - j * p.heads;
        const int first = (b0 + j) * p.block, old = max(0, n - first), end = min(p.block, n + count - first);
        int pg, slot;
        find_slot(p.view, b, first, &pg, &slot);
        const uint8_t* src = in.p + b * in.sb + head * in.sh;
#pragma unroll 1
        for (int c = l; c < N * L; c += L) {
          const int r = c / C;
          u32x2* to = (u32x2*)(pool.row(pg, head, slot + r) + 8 * (c % C));
          float f[8];
          double by = 1.0;
          if (r < old) {
            if (!(s > was)) continue;
            const u32x2 w = *to;
#pragma unroll
            for (int e = 0; e < 8; ++e) f[e] = (float)(int8_t)(w[e / 4] >> 8 * (e % 4));
            by = was;
          } else if (r < end) {
            Io<T>::unpack(((const u32x4*)(src + (int64_t)(first + r - n) * in.st))[c % C], f);
          } else {
            continue;
          }
          *to = codes8(f, by, s);
        }
      }
    }
  }
}

template <NormType T, int C, int L, int N, int M, bool STREAM>
hipError_t go(const AppendParams& p, int64_t tasks, hipStream_t s) {
  const int64_t per = (int64_t)kThreads / L * M;
  const dim3 grid((unsigned)std::min<int64_t>((tasks + per - 1) / per, 1 << 20), (unsigned)std::min(p.B, 65535), 2);
  hipLaunchKernelGGL((append_i8<T, C, L, N, M, STREAM>), grid, dim3(kThreads), 0, s, p);
  return hipGetLastError();
}

// Blocks of up to CHUNKS chunks. Where that makes three workgroups per CU, a thread has four
// chunks (two of the smallest blocks), of two tasks if need be: index arithmetic, maximum and
// scale are for all of a task's threads, and a chunk alone does not keep the memory busy. One
// chunk each is quicker for fewer. us, one chunk / so, 8 heads of 128: 8 sequences of 500 to 4000
// tokens, blocks of 1, 45.2 / 24.7, of 2 77 / 24.1, of 4 44.2 / 22.4; 2 of 1000 in blocks of 1
// 5.9 / 6.8, 8 of 500 10.3 / 7.2.
template <NormType T, int C, int CHUNKS> hipError_t run_append(const AppendParams& p, hipStream_t s) {
  const int64_t tasks = ((int64_t)p.T + 2 * p.block - 2) / p.block * p.heads;   // of a sequence, at most
  // (in floating point: broadcast rows may be any number)
  const bool stream = (double)p.B * p.T * p.heads * (C * 16) >= kStream;
  if constexpr (CHUNKS > 512) {
    constexpr int N = CHUNKS / 256;
    return stream ? go<T, C, 256, N, 1, true>(p, tasks, s) : go<T, C, 256, N, 1, false>(p, tasks, s);
  } else {
    constexpr int N = CHUNKS > 256 ? 8 : CHUNKS > 16 ? 4 : 2, L = CHUNKS / N, M = N == 2 ? 2 : 1;
    constexpr int few = CHUNKS < 64 ? CHUNKS : 64;
    if (stream) return go<T, C, L, N, M, true>(p, tasks, s);
    if (2.0 * p.B * tasks >= 3 * 256 * (kThreads / L * M)) return go<T, C, L, N, M, false>(p, tasks, s);
    return go<T, C, few, CHUNKS / few, 1, false>(p, tasks, s);
  }
}

template <NormType T, int C> hipError_t run_append(const AppendParams& p, hipStream_t s) {
  const int chunks = p.block * C;
  if constexpr (C == 8)
    if (chunks <= 8) return run_append<T, C, 8>(p, s);
  if (chunks <= 16) return run_append<T, C, 16>(p, s);
  if (chunks <= 32) return run_append<T, C, 32>(p, s);
  if (chunks <= 64) return run_append<T, C, 64>(p, s);
  if (chunks <= 128) return run_append<T, C, 128>(p, s);
  if (chunks <= 256) return run_append<T, C, 256>(p, s);
  if (chunks <= 512) return run_append<T, C, 512>(p, s);
  if (chunks <= 1024) return run_append<T, C, 1024>(p, s);
  if (chunks <= 2048) return run_append<T, C, 2048>(p, s);
  if (chunks <= 4096) return run_append<T, C, 4096>(p, s);
  return hipErrorNotSupported;
}

// ---- read --------------------------------------------------------------------

struct ReadParams {
  PagedView view;
  Pool8 pool[2];
  uint8_t* out[2];
  int64_t sb[2], sh[2], st[2];   // bytes
  const int* first;
  PageDiv by_T, by_block;
  int B, T, heads;
};

// 8 codes times their scale s, to memory; as fp32 the second four lie C pieces of 16 bytes behind
// the first, so that the threads of a row write neighbouring ones; `odd`: some of a wave's
// products may lie past the type's range, where they are its largest value, or s may be no number.
template <NormType T>
constexpr float kMost = T == NormType::F16 ? 65504.0f : T == NormType::BF16 ? 0x1.fep127f : __FLT_MAX__;
template <NormType T, int C, bool STREAM>
__device__ __forceinline__ void put8(uint8_t* to, u32x2 w, float s, bool odd) {
  float f[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) f[e] = (float)(int8_t)(w[e / 4] >> 8 * (e % 4)) * s;
  if (odd)
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = fminf(fmaxf(f[e], -kMost<T>), kMost<T>) + s * 0.0f;
#pragma unroll
  for (int i = 0; i < 8 / Io<T>::kVec; ++i) {
    const u32x4 x = Io<T>::pack(f + i * Io<T>::kVec);
    if constexpr (STREAM) __builtin_nontemporal_store(x, (u32x4*)to + i * C);
    else ((u32x4*)to)[i * C] = x;
  }
}

// U rows of a key and a value to a thread's chunk, all loaded before the first is stored; a
// head's rows follow one another, as outputs mostly lie. us, 8 sequences of 5000 to 8192 slots
// of 8 heads of 128 into bf16: 71.4 (5.3 TB/s, of which 72 % are writes); heads side by side 73,
// stores through the caches 78, loads through them 72.3, keys and values by different
// workgroups 75, 8 rows at a time 80. Into fp32 120 (5.2 TB/s); 4 rows at a time 125, a thread's
// eight values side by side, which leaves lines half written, 155. 3 sequences of 1001 to 1500
// slots of 64 5.4 (with 4 rows at a time 6.3).
constexpr int rows_of(NormType t, bool stream) { return stream && t != NormType::F32 ? 4 : 2; }
template <NormType T, int C, bool STREAM>
__global__ __launch_bounds__(kThreads) void read_i8(ReadParams p) {
  constexpr int R = kThreads / C, U = rows_of(T, STREAM);
  const int c = threadIdx.x % C, first = threadIdx.x / C;
  const int rows = p.T * p.heads;
  for (int b = blockIdx.y; b < p.B; b += gridDim.y) {
    const int len = clamp_length(p.view.lengths[b], p.view.room);
    const int64_t from = p.first ? max(0, p.first[b]) : 0;
    for (int64_t r0 = (int64_t)blockIdx.x * R * U; r0 < rows; r0 += (int64_t)gridDim.x * R * U) {
      u32x2 w[2][U];
      float s[2][U];
      int t[U], h[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int r = (int)min<int64_t>(r0 + u * R + first, rows - 1);
        h[u] = div_page(p.by_T, r);
        t[u] = r - h[u] * p.T;
        const int64_t slot = from + t[u];
        int page, row;
        const bool there = find_slot(p.view, b, (int)min<int64_t>(slot, max(len - 1, 0)), &page, &row) & (slot < len);
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          w[x][u] = u32x2{0, 0};
          s[x][u] = 0.0f;
          if (there) {
            const uint8_t* src = p.pool[x].row(page, h[u], row);
            if constexpr (T == NormType::F32) w[x][u] = u32x2{((const uint32_t*)src)[c], ((const uint32_t*)src)[C + c]};
            else if constexpr (STREAM) w[x][u] = __builtin_nontemporal_load((const u32x2*)src + c);
            else w[x][u] = ((const u32x2*)src)[c];
            s[x][u] = *p.pool[x].scale_of(page, h[u], div_page(p.by_block, row));
          }
        }
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (r0 + u * R + first >= rows) break;
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const bool odd = __ballot(!(fabsf(s[x][u]) <= kMost<T> / 128.0f)) != 0;
          uint8_t* to = p.out[x] + b * p.sb[x] + h[u] * p.sh[x] + t[u] * p.st[x];
          put8<T, C, STREAM>(to + 16 * c, w[x][u], s[x][u], odd);
        }
      }
    }
  }
}

template <NormType T, int C> hipError_t run_read(const ReadParams& p, hipStream_t s) {
  const int64_t rows = (int64_t)p.T * p.heads;
  const bool stream = p.B * rows * C * 16 >= kStream;
  const int64_t per = kThreads / C * rows_of(T, stream);
  const dim3 grid((unsigned)std::min<int64_t>((rows + per - 1) / per, 1 << 20), (unsigned)std::min(p.B, 65535));
  if (stream) hipLaunchKernelGGL((read_i8<T, C, true>), grid, dim3(kThreads), 0, s, p);
  else hipLaunchKernelGGL((read_i8<T, C, false>), grid, dim3(kThreads), 0, s, p);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_paged_append_i8(AttnType t, const PagedAppendDesc& d, const QuantScales& q, hipStream_t s) {
  AppendParams p{};
  p.view = view_of(d.c);
  p.pool[0] = pool_of(d.c, q, false);
  p.pool[1] = pool_of(d.c, q, true);
  p.rows[0] = {(const uint8_t*)d.k, 2 * d.k_sb, 2 * d.k_sh, 2 * d.k_st};
  p.rows[1] = {(const uint8_t*)d.v, 2 * d.v_sb, 2 * d.v_sh, 2 * d.v_st};
  p.counts = d.counts;
  p.by_heads = page_div(d.c.heads);
  p.by_block = page_div(q.block);
  p.B = d.c.B; p.T = d.T; p.heads = d.c.heads; p.block = q.block;
  if (t == AttnType::BF16) {
    if (d.c.D == 128) return run_append<NormType::BF16, 16>(p, s);
    if (d.c.D == 64) return run_append<NormType::BF16, 8>(p, s);
  } else {
    if (d.c.D == 128) return run_append<NormType::F16, 16>(p, s);
    if (d.c.D == 64) return run_append<NormType::F16, 8>(p, s);
  }
  return hipErrorNotSupported;
}

hipError_t launch_paged_read_i8(NormType t, const PagedReadDesc& d, const QuantScales& q, hipStream_t s) {
  ReadParams p{};
  const int size = t == NormType::F32 ? 4 : 2;
  p.view = view_of(d.c);
  p.pool[0] = pool_of(d.c, q, false);
  p.pool[1] = pool_of(d.c, q, true);
  p.out[0] = (uint8_t*)d.k; p.sb[0] = size * d.k_sb; p.sh[0] = size * d.k_sh; p.st[0] = size * d.k_st;
  p.out[1] = (uint8_t*)d.v; p.sb[1] = size * d.v_sb; p.sh[1] = size * d.v_sh; p.st[1] = size * d.v_st;
  p.first = d.first;
  p.by_T = page_div(d.T);
  p.by_block = page_div(q.block);
  p.B = d.c.B; p.T = d.T; p.heads = d.c.heads;
  if (d.c.D != 64 && d.c.D != 128) return hipErrorNotSupported;
  const bool wide = d.c.D == 128;
  switch (t) {
    case NormType::BF16: return wide ? run_read<NormType::BF16, 16>(p, s) : run_read<NormType::BF16, 8>(p, s);
    case NormType::F16:  return wide ? run_read<NormType::F16, 16>(p, s) : run_read<NormType::F16, 8>(p, s);
    case NormType::F32:  return wide ? run_read<NormType::F32, 16>(p, s) : run_read<NormType::F32, 8>(p, s);
  }
  return hipErrorNotSupported;
}

}  // namespace grxk
