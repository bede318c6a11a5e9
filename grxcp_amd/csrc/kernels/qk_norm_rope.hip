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
//    are computed once per token (into LDS) and not once per head;
//  * an angle is position * frequency in full: the product and its division by 2 pi are
//    64-bit with their remainders, so that position 10^6 and beyond turn by what the
//    formula says, and the part of a turn that is left goes through polynomials.

#include "../launch.h"
#include "device_common.h"
#include "paged_common.h"
#include "row_io.h"

#include <algorithm>

namespace grxk {
namespace {

constexpr int kThreads = 256, kWaves = kThreads / 64;
constexpr int kAngles = 1024;          // cosines of a workgroup's tokens

// Rows of [B, heads, S, D], strides in bytes.
struct Rows {
  uint8_t* p;
  int64_t sb, sh, ss;
  __device__ __forceinline__ uint8_t* at(int b, int h, int s) const { return p + b * sb + h * sh + s * ss; }
};

struct Part {                          // queries or keys
  Rows x, dy, y;                       // y: dx of a backward call
  const uint8_t* gamma;                // null: no norm
  int heads;
  PageDiv by_heads;
};

struct RParams {
  Part part[2];
  const int* positions;
  const float* inv_freq;
  float* partial;                      // [workgroups, 2, D], or null: no gradient of the gains
  PageDiv by_s;
  int S, tokens;
  int tile;                            // tokens of a workgroup's tile
  int tiles;
  int rotary;
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
  const float sx = fmaf(x * z, fmaf(z, fmaf(z, fmaf(z, 2.7557319e-6f, -1.9841270e-4f), 8.3333333e-3f), -1.6666667e-1f), x);
  const float cx = fmaf(z, fmaf(z, fmaf(z, fmaf(z, fmaf(z, -2.7557319e-7f, 2.4801587e-5f), -1.3888889e-3f), 4.1666667e-2f), -0.5f), 1.0f);
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

// 8 values at p.
template <NormType T> __device__ __forceinline__ void load8(const uint8_t* p, u32x4 (&w)[8 / Io<T>::kVec]) {
#pragma unroll
  for (int i = 0; i < 8 / Io<T>::kVec; ++i) w[i] = ((const u32x4*)p)[i];
}
template <NormType T> __device__ __forceinline__ void unpack8(const u32x4 (&w)[8 / Io<T>::kVec], float* f) {
#pragma unroll
  for (int i = 0; i < 8 / Io<T>::kVec; ++i) Io<T>::unpack(w[i], f + i * Io<T>::kVec);
}
template <NormType T> __device__ __forceinline__ void store8(uint8_t* p, const float* f) {
#pragma unroll
  for (int i = 0; i < 8 / Io<T>::kVec; ++i) ((u32x4*)p)[i] = Io<T>::pack(f + i * Io<T>::kVec);
}

template <NormType T, int D, bool PAIRS, bool BWD>
__global__ __launch_bounds__(kThreads) void qk_norm_rope(RParams p) {
  constexpr int G = D / 16, RW = 64 / G;   // lanes of a row, rows of a wave
  constexpr int W = 8 / Io<T>::kVec;
  constexpr int E = Io<T>::kVec == 8 ? 2 : 4;
  __shared__ __attribute__((aligned(16))) float cs[2][kAngles];
  __shared__ float red[BWD ? kWaves : 1][BWD ? 2 * D : 1];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int g = lane / G, l = lane % G;
  const int half = p.rotary / 2, rc = p.rotary / 16;
  // the lane's two chunks of 8 values
  int c0 = l, c1 = l + G;
  if constexpr (!PAIRS) {
    c0 = l < rc ? l : 2 * l;               // behind the rotated ones: 2 rc + 2 (l - rc)
    c1 = l < rc ? l + rc : 2 * l + 1;
  }
  float acc[2][16];
  if constexpr (BWD)
#pragma unroll
    for (int i = 0; i < 16; ++i) acc[0][i] = acc[1][i] = 0.0f;

  for (int t = blockIdx.x; t < p.tiles; t += gridDim.x) {
    const int t0 = t * p.tile, n = min(p.tile, p.tokens - t0);
    if (half) {
      __syncthreads();                     // the tile before has been read
      for (int i = tid; i < n * half; i += kThreads) {
        const int tok = i / half, f = i - tok * half;
        cos_sin(p.positions[t0 + tok], p.inv_freq[f], cs[0][i], cs[1][i]);
      }
      __syncthreads();
    }
    const int passes0 = (n * p.part[0].heads + RW - 1) / RW, passes = passes0 + (n * p.part[1].heads + RW - 1) / RW;
    for (int y = blockIdx.y * kWaves + wave; y < passes; y += gridDim.y * kWaves) {
      const int which = y >= passes0;
      const Part& q = p.part[which];
      const int r = (which ? y - passes0 : y) * RW + g;
      const bool live = r < n * q.heads;
      const int row = live ? r : 0;
      const int tok = div_page(q.by_heads, row), h = row - tok * q.heads;
      const int b = div_page(p.by_s, t0 + tok), s = t0 + tok - b * p.S;
      float x[2][8], d[2][8], gam[2][8], inv = 1.0f;
      u32x4 wx[2][W], wd[2][W], wg[2][W];
      const uint8_t* px = q.x.at(b, h, s);
      const bool norm = q.gamma != nullptr;
      if (!BWD || norm) {
        load8<T>(px + 8 * E * c0, wx[0]);
        load8<T>(px + 8 * E * c1, wx[1]);
      }
      if constexpr (BWD) {
        const uint8_t* pd = q.dy.at(b, h, s);
        load8<T>(pd + 8 * E * c0, wd[0]);
        load8<T>(pd + 8 * E * c1, wd[1]);
      }
      if (norm) {
        load8<T>(q.gamma + 8 * E * c0, wg[0]);
        load8<T>(q.gamma + 8 * E * c1, wg[1]);
      }
      if (!BWD || norm) {
        unpack8<T>(wx[0], x[0]);
        unpack8<T>(wx[1], x[1]);
      }
      if (norm) {
        unpack8<T>(wg[0], gam[0]);
        unpack8<T>(wg[1], gam[1]);
        float ss = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) ss = fmaf(x[0][i], x[0][i], fmaf(x[1][i], x[1][i], ss));
        inv = rsqrtf(fmaf(row_sum<G>(ss), 1.0f / D, p.eps));
      }
      if constexpr (BWD) {
        unpack8<T>(wd[0], d[0]);
        unpack8<T>(wd[1], d[1]);
      }
      // the row to rotate
      float (&v)[2][8] = BWD ? d : x;
      if constexpr (!BWD)
        if (norm)
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            v[0][i] = v[0][i] * inv * gam[0][i];
            v[1][i] = v[1][i] * inv * gam[1][i];
          }
      const float* co = cs[0] + tok * half;
      const float* si = cs[1] + tok * half;
      if constexpr (PAIRS) {
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const int at = c ? c1 : c0;
          if (at < 2 * rc)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const float cc = co[4 * at + i], sn = BWD ? -si[4 * at + i] : si[4 * at + i];
              const float a = v[c][2 * i], bb = v[c][2 * i + 1];
              v[c][2 * i] = fmaf(a, cc, -(bb * sn));
              v[c][2 * i + 1] = fmaf(bb, cc, a * sn);
            }
        }
      } else {
        if (l < rc)
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const float cc = co[8 * l + i], sn = BWD ? -si[8 * l + i] : si[8 * l + i];
            const float a = v[0][i], bb = v[1][i];
            v[0][i] = fmaf(a, cc, -(bb * sn));
            v[1][i] = fmaf(bb, cc, a * sn);
          }
      }
      if constexpr (BWD)
        if (norm) {
          float dot = 0.0f;
          float (&to)[16] = acc[0];
#pragma unroll
          for (int c = 0; c < 2; ++c)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              x[c][i] *= inv;              // n
              if (live) {
                if (which) acc[1][8 * c + i] = fmaf(d[c][i], x[c][i], acc[1][8 * c + i]);
                else to[8 * c + i] = fmaf(d[c][i], x[c][i], to[8 * c + i]);
              }
              d[c][i] *= gam[c][i];
              dot = fmaf(d[c][i], x[c][i], dot);
            }
          dot = row_sum<G>(dot) * (1.0f / D);
#pragma unroll
          for (int c = 0; c < 2; ++c)
#pragma unroll
            for (int i = 0; i < 8; ++i) d[c][i] = inv * fmaf(-x[c][i], dot, d[c][i]);
        }
      if (live) {
        uint8_t* to = q.y.at(b, h, s);
        store8<T>(to + 8 * E * c0, v[0]);
        store8<T>(to + 8 * E * c1, v[1]);
      }
    }
  }
  if constexpr (BWD) {
    if (!p.partial) return;
    // a wave's rows, then the workgroup's waves
#pragma unroll
    for (int w = 0; w < 2; ++w)
#pragma unroll
      for (int c = 0; c < 2; ++c)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          float v = acc[w][8 * c + i];
#pragma unroll
          for (int o = G; o < 64; o <<= 1) v += __shfl_xor(v, o);
          if (g == 0) red[wave][w * D + 8 * (c ? c1 : c0) + i] = v;
        }
    __syncthreads();
    float* out = p.partial + (int64_t)(blockIdx.y * gridDim.x + blockIdx.x) * 2 * D;
    for (int i = tid; i < 2 * D; i += kThreads) {
      float v = red[0][i];
#pragma unroll
      for (int w = 1; w < kWaves; ++w) v += red[w][i];
      out[i] = v;
    }
  }
}

// The gains' gradients from the workgroups' parts, 16 columns to a workgroup, in the same
// order every time.
__global__ __launch_bounds__(1024) void gain_grad(const float* partial, int parts, int D, float* dq, float* dk) {
  __shared__ float red[64][17];
  const int col = threadIdx.x & 15, lane = threadIdx.x >> 4, at = blockIdx.x * 16 + col;
  float v = 0.0f;
#pragma unroll 8
  for (int i = lane; i < parts; i += 64) v += partial[(int64_t)i * 2 * D + at];
  red[lane][col] = v;
  __syncthreads();
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    if (lane < o) red[lane][col] += red[lane + o][col];
    __syncthreads();
  }
  if (lane == 0) {
    float* out = at < D ? dq : dk;
    if (out) out[at < D ? at : at - D] = red[0][col];
  }
}

struct RopePlan {
  int tile, tiles, x, y;
};
RopePlan plan_of(int64_t tokens, int hq, int hk, int D, bool bwd) {
  RopePlan r{};
  const int rw = 64 / (D / 16), rows = kWaves * rw;   // rows of a pass of a wave, of a workgroup
  const int heads = hq + hk;
  // Few rows: a token to a workgroup, and its heads to several. Many: tokens enough for
  // their angles to keep the threads at work, and for four passes.
  r.tile = tokens * heads < 2048 * rows
               ? 1 : std::min({kAngles / (D / 2), 16, std::max(4, (4 * rows + heads - 1) / heads)});
  r.tiles = (int)((tokens + r.tile - 1) / r.tile);
  const int passes = (hq + rw - 1) / rw + (hk + rw - 1) / rw;
  r.y = r.tile > 1 ? 1 : std::min((passes + kWaves - 1) / kWaves, 8);
  r.x = (int)std::min<int64_t>(r.tiles, bwd ? std::max(1, 1024 / r.y) : (1 << 20));
  return r;
}

template <NormType T, int D> hipError_t run(const QkRopeDesc& d, bool bwd, hipStream_t s) {
  RParams p{};
  const int size = T == NormType::F32 ? 4 : 2;
  auto rows = [&](const QkRows& r) { return Rows{(uint8_t*)r.p, r.sb * size, r.sh * size, r.ss * size}; };
  bool gains = false;
  for (int i = 0; i < 2; ++i) {
    Part& q = p.part[i];
    q.heads = d.heads[i];
    q.by_heads = page_div(std::max(1, q.heads));
    if (!q.heads) continue;
    q.x = rows(d.x[i]);
    q.dy = rows(d.dy[i]);
    q.y = rows(d.y[i]);
    q.gamma = (const uint8_t*)d.gamma[i];
    gains |= d.dgamma[i] != nullptr;
  }
  p.positions = d.positions;
  p.inv_freq = d.inv_freq;
  p.rotary = d.rotary;
  p.eps = d.eps;
  p.S = d.S;
  p.by_s = page_div(std::max(1, d.S));
  p.tokens = d.B * d.S;
  if (p.tokens == 0 || d.heads[0] + d.heads[1] == 0) {   // sums over no rows
    hipLaunchKernelGGL(gain_grad, dim3(2 * D / 16), dim3(1024), 0, s, nullptr, 0, D, d.dgamma[0], d.dgamma[1]);
    return hipGetLastError();
  }
  const RopePlan r = plan_of(p.tokens, d.heads[0], d.heads[1], D, bwd);
  p.tile = r.tile;
  p.tiles = r.tiles;
  p.partial = bwd && gains ? (float*)d.ws : nullptr;
  const dim3 grid(r.x, r.y), threads(kThreads);
  auto go = [&](auto kern) { hipLaunchKernelGGL(kern, grid, threads, 0, s, p); };
  if (bwd) {
    if (d.pairs) go(qk_norm_rope<T, D, true, true>);
    else go(qk_norm_rope<T, D, false, true>);
  } else {
    if (d.pairs) go(qk_norm_rope<T, D, true, false>);
    else go(qk_norm_rope<T, D, false, false>);
  }
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess || !p.partial) return e;
  hipLaunchKernelGGL(gain_grad, dim3(2 * D / 16), dim3(1024), 0, s, p.partial, r.x * r.y, D, d.dgamma[0], d.dgamma[1]);
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
  return (size_t)r.x * r.y * 2 * D * sizeof(float);
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
