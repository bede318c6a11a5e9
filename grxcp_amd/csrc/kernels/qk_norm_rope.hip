// grxDNN norm and rotation of queries and keys, each head's row by itself, forward and
// backward, on gfx950.
//
// New: the reference plans normalisation and attention for grxDNN (ref
// docs/designs/grxcp_roadmap.md:864-877) and ships neither.
//
// With n = x r, r = 1 / sqrt(mean x^2 + eps), and R the rotation by the token's angles,
//   y  = R (n gamma)
//   g  = R^T dy,  dgamma = sum over rows of g n,  dx = r (g gamma - n mean(g gamma n)).
// Every value is read and written once, so both are bound by memory. What carries that:
//
//  * a row is held by D / 16 lanes, 16 values each, chosen so that both values of a
//    rotated pair are in one lane: chunks p and p + R / 16 where the halves of a row
//    pair up, any two chunks where neighbours do. A row's sums stay within 16 lanes;
//  * a workgroup takes a few tokens with all of their heads, so that cosines and sines
//    are computed once per token (into LDS) and not once per head. A backward call's
//    workgroups take queries or keys, and keep the sums of their gains in registers;
//  * what does not fit the caches is loaded and stored past them, two passes at a time, in
//    whole lines of 128 bytes. Where a lane's chunks are not that (rows of 64, fp32, halves that
//    turn only a part of the row) they go through LDS. us, direct / so, 16384 tokens of 40 heads
//    of 128 bf16 of which 32 turn 85 / 60, of 64 39.7 / 33.8, 24 heads of 128 fp32 84 / 72; backward
//    109 / 93.6, 59.6 / 53.5, 124 / 114. Whole lines already (128 bf16) 59.6 / 59.8, backward
//    97.3 / 100, and through the caches, which put lines together (6000 tokens of 40 heads of 64)
//    12.2 / 12.9.
//    Every angle, sum and product left out makes 1 % of a difference (61.5 to 60.9 us at
//    16384 tokens of 40 heads of 128): the order of loads and stores is what counts.
//    Queries and keys by different workgroups in the forward call took 71 for 60;
//  * an angle is position * frequency in full: the product and its division by 2 pi are
//    64-bit with their remainders, so that position 10^6 and beyond turn by what the
//    formula says, and the part of a turn that is left goes through polynomials.

#include "../launch.h"
#include "device_common.h"
#include "paged_common.h"
#include "row_io.h"

#include <algorithm>
#include <type_traits>

namespace grxk {
namespace {

constexpr int kThreads = 256, kWaves = kThreads / 64;
constexpr int kAngles = 1024;          // cosines of a workgroup's tokens
constexpr int kBackward = 768;         // workgroups of a backward call: three per CU, as its registers allow
constexpr int64_t kStream = 48 << 20;  // bytes from which on values are not kept in the caches

// Rows of [B, heads, S, D], strides in bytes.
struct Rows {
  uint8_t* p;
  int64_t sb, sh, ss;
  __device__ __forceinline__ uint8_t* at(int b, int h, int s) const { return p + b * sb + h * sh + s * ss; }
};

struct Part {                          // queries or keys
  Rows x, dy, y;                       // y: dx of a backward call
  const uint8_t* gamma;
  int heads;
  PageDiv by_heads;
};

// The workgroups that share one list of tiles: of both parts together in a forward call,
// of each part in a backward one.
struct Group {
  int tile, tiles;                     // tokens of a workgroup's tile
  int first, wgs;                      // its workgroups
};

struct RParams {
  Part part[2];
  Group group[2];
  const int* positions;
  const float* inv_freq;
  float* partial;                      // [workgroups, D], or null: no gradient of the gains
  PageDiv by_s, by_half;
  int S, tokens;
  int rotary;
  int norm;                            // 0: rotation alone
  float eps;
};

// cos and sin of position * f (|position * f| < 2^40).
__device__ __forceinline__ void cos_sin(int position, float f, float& c, float& s) {
  constexpr double kTurn = 0x1.45f306dc9c883p-3, kTurnLo = -0x1.6b01ec5417056p-57;   // 1 / (2 pi)
  const double a = (double)position * (double)f;
  const double e = fma((double)position, (double)f, -a);
  const double n = rint(a * kTurn);
  const double u = fma(a, kTurn, -n) + fma(a, kTurnLo, e * kTurn);   // of a turn
  const double q = rint(4.0 * u);
  const float x = (float)(u - 0.25 * q) * 6.28318530717958648f;      // -pi/4 .. pi/4
  const float z = x * x;
  // Taylor: the first terms left out are below 2^-28
  const float s3 = fmaf(z, fmaf(z, fmaf(z, 2.7557319e-6f, -1.9841270e-4f), 8.3333333e-3f), -1.6666667e-1f);
  const float sx = fmaf(x * z, s3, x);
  const float c4 = fmaf(z, fmaf(z, fmaf(z, -2.7557319e-7f, 2.4801587e-5f), -1.3888889e-3f), 4.1666667e-2f);
  const float cx = fmaf(z, fmaf(z, c4, -0.5f), 1.0f);
  const int k = (int)q & 3;
  const float a0 = (k & 1) ? sx : cx, b0 = (k & 1) ? cx : sx;
  c = (k == 1 || k == 2) ? -a0 : a0;
  s = (k >= 2) ? -b0 : b0;
}

// Sum over the G lanes (4, 8 or 16, neighbours) of a row, the same in each.
template <int G> __device__ __forceinline__ float row_sum(float v) {
#pragma clang fp contract(off)
  v += dpp_f<0xb1>(v);
  v += dpp_f<0x4e>(v);
  if constexpr (G >= 8) v += dpp_f<0x141>(v);
  if constexpr (G >= 16) v += dpp_f<0x140>(v);
  return v;
}

template <bool STREAM> __device__ __forceinline__ u32x4 load1(const uint8_t* p) {
  if constexpr (STREAM) return __builtin_nontemporal_load((const u32x4*)p);
  else return *(const u32x4*)p;
}
template <bool STREAM> __device__ __forceinline__ void store1(uint8_t* p, u32x4 w) {
  if constexpr (STREAM) __builtin_nontemporal_store(w, (u32x4*)p);
  else *(u32x4*)p = w;
}
// 8 values at p.
template <NormType T, bool STREAM>
__device__ __forceinline__ void load8(const uint8_t* p, u32x4 (&w)[8 / Io<T>::kVec]) {
#pragma unroll
  for (int i = 0; i < 8 / Io<T>::kVec; ++i) w[i] = load1<STREAM>(p + 16 * i);
}
template <NormType T> __device__ __forceinline__ void unpack8(const u32x4 (&w)[8 / Io<T>::kVec], float* f) {
#pragma unroll
  for (int i = 0; i < 8 / Io<T>::kVec; ++i) Io<T>::unpack(w[i], f + i * Io<T>::kVec);
}
template <NormType T> __device__ __forceinline__ void pack8(const float* f, u32x4 (&w)[8 / Io<T>::kVec]) {
#pragma unroll
  for (int i = 0; i < 8 / Io<T>::kVec; ++i) w[i] = Io<T>::pack(f + i * Io<T>::kVec);
}
template <NormType T, bool STREAM> __device__ __forceinline__ void store8(uint8_t* p, const float* f) {
  u32x4 w[8 / Io<T>::kVec];
  pack8<T>(f, w);
#pragma unroll
  for (int i = 0; i < 8 / Io<T>::kVec; ++i) store1<STREAM>(p + 16 * i, w[i]);
}

template <NormType T, int D, bool PAIRS, bool BWD, bool STREAM, bool LINES>
__global__ __launch_bounds__(kThreads, BWD ? 3 : 1) void qk_norm_rope(RParams p) {
  constexpr int G = D / 16, RW = 64 / G;   // lanes of a row, rows of a wave
  constexpr int W = 8 / Io<T>::kVec;
  constexpr int E = Io<T>::kVec == 8 ? 2 : 4;
  constexpr int U = BWD ? (Io<T>::kVec == 8 ? 2 : 1) : STREAM ? 2 : 1;   // passes at a time
  __shared__ __attribute__((aligned(16))) float cs[2][kAngles];
  __shared__ float red[BWD ? kWaves : 1][BWD ? D : 1];
  // LINES: a pass's rows lie here between memory, where a load takes whole rows, and the lanes
  constexpr int PR = D * E / 16, PC = 2 * W;   // 16-byte pieces of a row, of a lane
  __shared__ __attribute__((aligned(16))) uint8_t stage[LINES ? kWaves : 1][LINES ? 64 * 16 * PC : 16];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int g = lane / G, l = lane % G;
  const int half = p.rotary / 2, rc = p.rotary / 16;
  const int own = BWD && (int)blockIdx.x >= p.group[1].first;   // the part of a backward call's workgroup
  const Group& gr = p.group[own];
  const bool norm = p.norm;
  // the lane's two chunks of 8 values
  int c0 = l, c1 = l + G;
  if constexpr (!PAIRS) {
    c0 = l < rc ? l : l + rc;              // behind the rotated ones: 2 rc + l - rc
    c1 = l < rc ? l + rc : l + G;
  }
  const int o0 = 8 * E * c0, o1 = 8 * E * c1;
  // A lane's pieces of the pass's rows as they lie in memory against its two chunks: in, or back.
  auto turn = [&](u32x4 (&w)[2][W], bool in) __attribute__((always_inline)) {
    uint8_t* rows = stage[LINES ? wave : 0];
    u32x4* lines = (u32x4*)rows + lane;
    u32x4* chunks[2] = {(u32x4*)(rows + g * D * E + o0), (u32x4*)(rows + g * D * E + o1)};
    if (in) {
#pragma unroll
      for (int k = 0; k < PC; ++k) lines[64 * k] = w[k / W][k % W];
    } else {
#pragma unroll
      for (int k = 0; k < PC; ++k) chunks[k / W][k % W] = w[k / W][k % W];
    }
    wave_fence();
    if (in) {
#pragma unroll
      for (int k = 0; k < PC; ++k) w[k / W][k % W] = chunks[k / W][k % W];
    } else {
#pragma unroll
      for (int k = 0; k < PC; ++k) w[k / W][k % W] = lines[64 * k];
    }
    wave_fence();
  };
  float acc[2][8];
#pragma unroll
  for (int i = 0; i < 8; ++i) acc[0][i] = acc[1][i] = 0.0f;
  u32x4 wg[2][W];                          // the gains
  if (BWD && norm) {
    load8<T, false>(p.part[own].gamma + o0, wg[0]);
    load8<T, false>(p.part[own].gamma + o1, wg[1]);
  }
  const int w = blockIdx.y * kWaves + wave, waves = kWaves * gridDim.y;

  for (int t = blockIdx.x - gr.first; t < gr.tiles; t += gr.wgs) {
    const int t0 = t * gr.tile, n = min(gr.tile, p.tokens - t0);
    if (half) {
      __syncthreads();                     // the tile before has been read
      for (int i = tid; i < n * half; i += kThreads) {
        const int tok = div_page(p.by_half, i), f = i - tok * half;
        cos_sin(p.positions[t0 + tok], p.inv_freq[f], cs[0][i], cs[1][i]);
      }
      __syncthreads();
    }
    // passes of RW rows each: the queries', then the keys'
    const int passes0 = BWD && own ? 0 : (n * p.part[0].heads + RW - 1) / RW;
    const int passes = BWD && !own ? passes0 : passes0 + (n * p.part[1].heads + RW - 1) / RW;
    for (int first = w; first < passes; first += U * waves) {
      // U passes' rows are asked for before the first is waited for
      u32x4 wx[U][2][W], wd[U][2][W];
      int64_t yo[U][LINES ? PC : 1];
      int toks[U];
      bool lives[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int pass = first + u * waves;
        if (pass >= passes) break;
        const int which = BWD ? own : pass >= passes0;
        const Part& q = p.part[which];
        const int r = (which && !BWD ? pass - passes0 : pass) * RW + g, rows = n * q.heads;
        lives[u] = r < rows;
        const int row = min(r, rows - 1);
        toks[u] = div_page(q.by_heads, row);
        if constexpr (LINES) {
#pragma unroll
          for (int k = 0; k < PC; ++k) {
            const int at = min(r - g + (64 * k + lane) / PR, rows - 1), piece = 16 * (lane % PR);
            const int tok = div_page(q.by_heads, at), h = at - tok * q.heads;
            const int b = div_page(p.by_s, t0 + tok), s = t0 + tok - b * p.S;
            if (!BWD || norm) wx[u][k / W][k % W] = load1<STREAM>(q.x.at(b, h, s) + piece);
            if constexpr (BWD) wd[u][k / W][k % W] = load1<STREAM>(q.dy.at(b, h, s) + piece);
            yo[u][k] = b * q.y.sb + h * q.y.sh + s * q.y.ss + piece;
          }
          continue;
        }
        const int h = row - toks[u] * q.heads;
        const int b = div_page(p.by_s, t0 + toks[u]), s = t0 + toks[u] - b * p.S;
        if (!BWD || norm) {
          const uint8_t* px = q.x.at(b, h, s);
          load8<T, STREAM>(px + o0, wx[u][0]);
          load8<T, STREAM>(px + o1, wx[u][1]);
        }
        if constexpr (BWD) {
          const uint8_t* pd = q.dy.at(b, h, s);
          load8<T, STREAM>(pd + o0, wd[u][0]);
          load8<T, STREAM>(pd + o1, wd[u][1]);
        }
        yo[u][0] = b * q.y.sb + h * q.y.sh + s * q.y.ss;
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (first + u * waves >= passes) break;
        const Part& q = p.part[BWD ? own : first + u * waves >= passes0];
        const int tok = toks[u];
        if constexpr (!BWD)
          if (norm) {
            load8<T, false>(q.gamma + o0, wg[0]);
            load8<T, false>(q.gamma + o1, wg[1]);
          }
        // cosines and sines of the lane's 8 pairs (those of lanes behind the turned values are not used)
        float co[8], si[8];
        if (half) {
          const int c = tok * half;
          if constexpr (PAIRS) {
            *(f32x4*)co = *(const f32x4*)&cs[0][c + min(4 * c0, half - 4)];
            *(f32x4*)(co + 4) = *(const f32x4*)&cs[0][c + min(4 * c1, half - 4)];
            *(f32x4*)si = *(const f32x4*)&cs[1][c + min(4 * c0, half - 4)];
            *(f32x4*)(si + 4) = *(const f32x4*)&cs[1][c + min(4 * c1, half - 4)];
          } else {
            const int k = c + min(8 * l, half - 8);
            *(f32x4*)co = *(const f32x4*)&cs[0][k];
            *(f32x4*)(co + 4) = *(const f32x4*)&cs[0][k + 4];
            *(f32x4*)si = *(const f32x4*)&cs[1][k];
            *(f32x4*)(si + 4) = *(const f32x4*)&cs[1][k + 4];
          }
        }
        if constexpr (LINES) {
          if (!BWD || norm) turn(wx[u], true);
          if constexpr (BWD) turn(wd[u], true);
        }
        if (lives[u]) {                      // (whole rows: the others' sums are their own)
          float x[2][8], d[2][8], inv = 1.0f;
          if (!BWD || norm) {
            unpack8<T>(wx[u][0], x[0]);
            unpack8<T>(wx[u][1], x[1]);
          }
          if (norm) {
            float ss = 0.0f;
#pragma unroll
            for (int i = 0; i < 8; ++i) ss = fmaf(x[0][i], x[0][i], fmaf(x[1][i], x[1][i], ss));
            inv = __builtin_amdgcn_rsqf(fmaf(row_sum<G>(ss), 1.0f / D, p.eps));
          }
          if constexpr (BWD) {
            unpack8<T>(wd[u][0], d[0]);
            unpack8<T>(wd[u][1], d[1]);
          }
          float gam[2][8];
          if (norm) {
            unpack8<T>(wg[0], gam[0]);
            unpack8<T>(wg[1], gam[1]);
          }
          float (&v)[2][8] = BWD ? d : x;      // what is turned
          if constexpr (!BWD)
            if (norm)
#pragma unroll
              for (int i = 0; i < 8; ++i) {
                v[0][i] = v[0][i] * inv * gam[0][i];   // (inv * gam may be past fp32)
                v[1][i] = v[1][i] * inv * gam[1][i];
              }
          if constexpr (PAIRS) {
#pragma unroll
            for (int c = 0; c < 2; ++c)
              if ((c ? c1 : c0) < 2 * rc)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                  const float a = v[c][2 * i], b = v[c][2 * i + 1];
                  const float k = co[4 * c + i], m = BWD ? -si[4 * c + i] : si[4 * c + i];
                  v[c][2 * i] = fmaf(a, k, -(b * m));
                  v[c][2 * i + 1] = fmaf(b, k, a * m);
                }
          } else {
            if (l < rc)
#pragma unroll
              for (int i = 0; i < 8; ++i) {
                const float a = v[0][i], b = v[1][i];
                const float m = BWD ? -si[i] : si[i];
                v[0][i] = fmaf(a, co[i], -(b * m));
                v[1][i] = fmaf(b, co[i], a * m);
              }
          }
          if constexpr (BWD)
            if (norm) {
              // with u = r g: dgamma += u x, dx = u gamma - x r^2 mean(u gamma x)
              float dot = 0.0f;
#pragma unroll
              for (int c = 0; c < 2; ++c)
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                  d[c][i] *= inv;
                  acc[c][i] = fmaf(d[c][i], x[c][i], acc[c][i]);
                  d[c][i] *= gam[c][i];
                  dot = fmaf(d[c][i], x[c][i], dot);
                }
              dot = row_sum<G>(dot) * (1.0f / D);
              const float by = inv * inv * dot;
              if (!(fabsf(by) <= __FLT_MAX__)) {   // (eps 0 and tiny rows, or no numbers)
#pragma unroll
                for (int c = 0; c < 2; ++c)
#pragma unroll
                  for (int i = 0; i < 8; ++i) d[c][i] = fmaf(-(x[c][i] * inv), inv * dot, d[c][i]);
              } else {
#pragma unroll
                for (int c = 0; c < 2; ++c)
#pragma unroll
                  for (int i = 0; i < 8; ++i) d[c][i] = fmaf(-x[c][i], by, d[c][i]);
              }
            }
          if constexpr (!LINES) {
            uint8_t* py = q.y.p + yo[u][0];
            store8<T, STREAM>(py + o0, v[0]);
            store8<T, STREAM>(py + o1, v[1]);
          } else {
            pack8<T>(v[0], wx[u][0]);
            pack8<T>(v[1], wx[u][1]);
          }
        }
        if constexpr (LINES) {
          turn(wx[u], false);
          const int r0 = (BWD || first + u * waves < passes0 ? first + u * waves : first + u * waves - passes0) * RW;
          const int rows = n * q.heads;
#pragma unroll
          for (int k = 0; k < PC; ++k)
            if (r0 + (64 * k + lane) / PR < rows) store1<STREAM>(q.y.p + yo[u][k], wx[u][k / W][k % W]);
        }
      }
    }
  }
  if constexpr (BWD) {
    if (!p.partial) return;
    // a wave's rows, then the workgroup's waves
#pragma unroll
    for (int c = 0; c < 2; ++c)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        float v = acc[c][i];
#pragma unroll
        for (int o = G; o < 64; o <<= 1) v += __shfl_xor(v, o);
        if (g == 0) red[wave][8 * (c ? c1 : c0) + i] = v;
      }
    __syncthreads();
    float* out = p.partial + (int64_t)(blockIdx.x * gridDim.y + blockIdx.y) * D;
    for (int i = tid; i < D; i += kThreads) {
      float v = red[0][i];
#pragma unroll
      for (int w = 1; w < kWaves; ++w) v += red[w][i];
      out[i] = v;
    }
  }
}

// The gains' gradients from the workgroups' parts (`nq` of the queries, then `nk` of the
// keys), 16 columns to a workgroup, in the same order every time.
__global__ __launch_bounds__(1024) void gain_grad(const float* partial, int nq, int nk, int D, float* dq, float* dk) {
  constexpr int kAtOnce = 16;
  __shared__ float red[16][16];
  const int col = threadIdx.x & 15, lane = threadIdx.x >> 4;
  const bool keys = (int)blockIdx.x * 16 >= D;
  const int at = blockIdx.x * 16 + col - (keys ? D : 0), n = keys ? nk : nq;
  float* out = keys ? dk : dq;
  if (!out) return;
  const float* from = partial + (keys ? (int64_t)nq * D : 0) + at;
  float v = 0.0f;
  for (int i = lane; i < n; i += 64 * kAtOnce) {
    float a[kAtOnce];
#pragma unroll
    for (int u = 0; u < kAtOnce; ++u) a[u] = from[(int64_t)min(i + 64 * u, n - 1) * D];
#pragma unroll
    for (int u = 0; u < kAtOnce; ++u) v += i + 64 * u < n ? a[u] : 0.0f;
  }
  v += __shfl_xor(v, 16);
  v += __shfl_xor(v, 32);
  if ((threadIdx.x & 63) < 16) red[threadIdx.x >> 6][col] = v;
  __syncthreads();
  if (threadIdx.x >= 16) return;
  v = 0.0f;
#pragma unroll
  for (int w = 0; w < 16; ++w) v += red[w][col];
  out[at] = v;
}

struct RopePlan {
  Group group[2];
  int y;
};
RopePlan plan_of(int64_t tokens, int hq, int hk, int D, bool bwd) {
  RopePlan r{};
  const int rw = 64 / (D / 16), rows = kWaves * rw;   // rows of a pass of a wave, of a workgroup
  // Few rows: a pass to a workgroup. Many: tokens enough for their angles to keep the threads
  // at work, and for four passes. us, few / many: 1600 tokens of 40 heads of 128 bf16 8.7 /
  // 9.1, 3003 of 32 of 64 fp32 10.9 / 9.9, 3200 of 40 of 128 14.6 / 12.4; backward, 3200 of
  // 40 26.3 / 28.6, 324 of 54 of 256 16.7 / 19.4.
  const bool few = tokens * (hq + hk) < (bwd ? 4096 : 1024) * rows;
  const int heads[2] = {bwd ? hq : hq + hk, bwd ? hk : 0};
  r.y = 1;
  for (int i = 0; i < 2; ++i) {
    Group& x = r.group[i];
    if (i) x.first = r.group[0].wgs;
    if (!heads[i]) continue;
    x.tile = std::min({few ? std::max(1, rows / heads[i]) : std::max(4, (4 * rows + heads[i] - 1) / heads[i]), 16,
                      kAngles / (D / 2)});
    x.tiles = (int)((tokens + x.tile - 1) / x.tile);
    if (few) r.y = std::max(r.y, std::min((heads[i] + rows - 1) / rows + !bwd, 8));
  }
  for (int i = 0; i < 2; ++i) {
    const int64_t most = bwd ? std::max<int64_t>(1, (int64_t)kBackward * heads[i] / (hq + hk) / r.y) : 1 << 20;
    r.group[i].wgs = (int)std::min<int64_t>(r.group[i].tiles, most);
  }
  r.group[1].first = r.group[0].wgs;
  return r;
}

template <NormType T, int D> hipError_t run(const QkRopeDesc& d, bool bwd, hipStream_t s) {
  RParams p{};
  const int size = T == NormType::F32 ? 4 : 2;
  auto rows = [&](const QkRows& r) { return Rows{(uint8_t*)r.p, r.sb * size, r.sh * size, r.ss * size}; };
  const bool gains = d.dgamma[0] || d.dgamma[1];
  for (int i = 0; i < 2; ++i) {
    Part& q = p.part[i];
    q.heads = d.heads[i];
    q.by_heads = page_div(std::max(1, q.heads));
    if (!q.heads) continue;
    q.x = rows(d.x[i]);
    q.dy = rows(d.dy[i]);
    q.y = rows(d.y[i]);
    q.gamma = (const uint8_t*)d.gamma[i];
    p.norm |= d.gamma[i] != nullptr;
  }
  p.positions = d.positions;
  p.inv_freq = d.inv_freq;
  p.rotary = d.rotary;
  p.by_half = page_div(std::max(1, d.rotary / 2));
  p.eps = d.eps;
  p.S = d.S;
  p.by_s = page_div(std::max(1, d.S));
  p.tokens = d.B * d.S;
  const RopePlan r =
      p.tokens && d.heads[0] + d.heads[1] ? plan_of(p.tokens, d.heads[0], d.heads[1], D, bwd) : RopePlan{};
  p.group[0] = r.group[0];
  p.group[1] = r.group[1];
  p.partial = bwd && gains ? (float*)d.ws : nullptr;
  const bool stream = (int64_t)p.tokens * (d.heads[0] + d.heads[1]) * D * size >= kStream;
  if (r.group[0].wgs + r.group[1].wgs) {
    const dim3 grid(r.group[0].wgs + r.group[1].wgs, r.y), threads(kThreads);
    auto go = [&](auto kern) { hipLaunchKernelGGL(kern, grid, threads, 0, s, p); };
    auto pick = [&](auto st, auto li) {
      constexpr bool ST = decltype(st)::value, LI = decltype(li)::value;
      if (bwd) {
        if (d.pairs) go(qk_norm_rope<T, D, true, true, ST, LI>);
        else go(qk_norm_rope<T, D, false, true, ST, LI>);
      } else {
        if (d.pairs) go(qk_norm_rope<T, D, true, false, ST, LI>);
        else go(qk_norm_rope<T, D, false, false, ST, LI>);
      }
    };
    const std::integral_constant<bool, true> yes;
    const std::integral_constant<bool, false> no;
    // Whether a lane's loads and stores are of whole lines by themselves.
    constexpr bool wide = T != NormType::F32 && D >= 128;
    if (!stream) {
      pick(no, no);
    } else if constexpr (wide) {
      if (d.pairs || d.rotary == D || d.rotary == 0) pick(yes, no);
      else pick(yes, yes);
    } else {
      pick(yes, yes);
    }
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  if (!bwd || !gains) return hipSuccess;
  hipLaunchKernelGGL(gain_grad, dim3(2 * D / 16), dim3(1024), 0, s, p.partial, r.group[0].wgs * r.y,
                     r.group[1].wgs * r.y, D, d.dgamma[0], d.dgamma[1]);
  return hipGetLastError();
}

template <NormType T> hipError_t run_d(const QkRopeDesc& d, bool bwd, hipStream_t s) {
  switch (d.D) {
    case 64:  return run<T, 64>(d, bwd, s);
    case 128: return run<T, 128>(d, bwd, s);
    case 256: return run<T, 256>(d, bwd, s);
  }
  return hipErrorNotSupported;
}

}  // namespace

size_t qk_norm_rope_workspace(int64_t tokens, int hq, int hk, int D) {
  const RopePlan r = plan_of(tokens, hq, hk, D, true);
  return (size_t)(r.group[0].wgs + r.group[1].wgs) * r.y * D * sizeof(float);
}

hipError_t launch_qk_norm_rope(NormType t, const QkRopeDesc& d, bool backward, hipStream_t s) {
  switch (t) {
    case NormType::BF16: return run_d<NormType::BF16>(d, backward, s);
    case NormType::F16:  return run_d<NormType::F16>(d, backward, s);
    case NormType::F32:  return run_d<NormType::F32>(d, backward, s);
  }
  return hipErrorNotSupported;
}

}  // namespace grxk
