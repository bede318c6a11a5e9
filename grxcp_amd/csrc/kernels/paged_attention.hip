// grxDNN attention of one new token per sequence over a paged key-value cache, on
// gfx950.
//
// New: the reference plans attention for grxDNN (ref
// docs/designs/grxcp_roadmap.md:864-877) and ships no code.

#include "../launch.h"
#include "device_common.h"
#include "paged_common.h"

#include <algorithm>

namespace grxk {
namespace {

template <AttnType T> struct PIo;
template <> struct PIo<AttnType::BF16> {
  __device__ static float ld(uint16_t b) { return bf16_to_f32(b); }
  __device__ static uint16_t st(float f) { return f32_to_bf16(f); }
};
template <> struct PIo<AttnType::F16> {
  __device__ static float ld(uint16_t b) { return f16_to_f32(b); }
  __device__ static uint16_t st(float f) { return f32_to_f16(f); }
};

struct DParams {
  PagedView view;
  const uint16_t* k; int64_t k_sp, k_sh, k_ss;
  const uint16_t* v; int64_t v_sp, v_sh, v_ss;
  const uint16_t* q; int64_t q_sb, q_sh;
  uint16_t* o; int64_t o_sb, o_sh;
  float* w; int64_t w_sb, w_sh;
  float decay;
  float* scores;      // [B, H, slots]
  float* stat;        // [B, H, 2]: maximum and sum
  int64_t slots;
  int B, H, heads, group;
  float c;            // scale * log2(e)
};

// One workgroup per query head: each of its four waves takes every fourth slot, a
// lane D / 64 values of a row, and the waves' results meet in LDS.
template <AttnType T, int D>
__global__ __launch_bounds__(256) void decode_heads(DParams p) {
  using IO = PIo<T>;
  constexpr int V = D / 64;
  __shared__ float part[4][D + 2];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int b = blockIdx.x / p.H, hq = blockIdx.x - b * p.H, h = hq / p.group;
  const int n = clamp_length(p.view.lengths[b], p.view.room);
  float q[V], acc[V], m = -INFINITY, l = 0.0f;
  for (int e = 0; e < V; ++e) {
    q[e] = IO::ld(p.q[b * p.q_sb + hq * p.q_sh + V * lane + e]);
    acc[e] = 0.0f;
  }
  float* scores = p.scores ? p.scores + blockIdx.x * p.slots : nullptr;
  for (int j = wave; j < n; j += 4) {
    int page, row;
    const bool there = find_slot(p.view, b, j, &page, &row);
    float s = -INFINITY;
    if (there) {
      const uint16_t* kr = p.k + page * p.k_sp + h * p.k_sh + row * p.k_ss + V * lane;
      const uint16_t* vr = p.v + page * p.v_sp + h * p.v_sh + row * p.v_ss + V * lane;
      s = 0.0f;
      for (int e = 0; e < V; ++e) s = fmaf(q[e], IO::ld(kr[e]), s);
      s = wave_sum(s) * p.c;
      const float top = fmaxf(fmaxf(m, s), -__FLT_MAX__);
      const float old = exp2f(m - top), w = exp2f(s - top);
      m = top;
      l = l * old + w;
      for (int e = 0; e < V; ++e) acc[e] = acc[e] * old + w * IO::ld(vr[e]);
    }
    if (scores && lane == 0) scores[j] = there ? s : INFINITY;   // +inf: no such slot
  }
  for (int e = 0; e < V; ++e) part[wave][V * lane + e] = acc[e];
  if (lane == 0) {
    part[wave][D] = m;
    part[wave][D + 1] = l;
  }
  __syncthreads();
  float top = -INFINITY, sum = 0.0f;
  for (int i = 0; i < 4; ++i) top = fmaxf(top, part[i][D]);
  const bool none = top == -INFINITY;       // no slot
  if (none) top = 0.0f;
  for (int i = 0; i < 4; ++i) sum += part[i][D + 1] * exp2f(part[i][D] - top);
  for (int d = threadIdx.x; d < D; d += 256) {
    float a = 0.0f;
    for (int i = 0; i < 4; ++i) a += part[i][d] * exp2f(part[i][D] - top);
    p.o[b * p.o_sb + hq * p.o_sh + d] = IO::st(none ? 0.0f : a / sum);
  }
  if (p.stat && threadIdx.x == 0) {
    p.stat[2 * blockIdx.x] = top;
    p.stat[2 * blockIdx.x + 1] = sum;
  }
}

// The slots' weights from the scores of a group's query heads.
__global__ __launch_bounds__(256) void slot_weights(DParams p) {
  const int b = blockIdx.y / p.heads, h = blockIdx.y - b * p.heads;
  const int n = clamp_length(p.view.lengths[b], p.view.room);
  float* w = p.w + b * p.w_sb + h * p.w_sh;
  for (int j = blockIdx.x * 256 + threadIdx.x; j < n; j += gridDim.x * 256) {
    float a = 0.0f;
    for (int i = 0; i < p.group; ++i) {
      const int64_t r = (int64_t)b * p.H + h * p.group + i;
      const float s = p.scores[r * p.slots + j];
      if (s != INFINITY) a += exp2f(s - p.stat[2 * r]) / p.stat[2 * r + 1];
    }
    w[j] = p.decay == 0.0f ? a : fmaf(p.decay, w[j], a);
  }
}

int64_t round_slots(int W, int page) { return ((int64_t)W * page + 127) / 128 * 128; }

template <AttnType T, int D>
hipError_t run(const PagedAttnDesc& d, hipStream_t s) {
  DParams p{};
  p.view = {d.c.table, d.c.table_rs, d.c.lengths, d.c.pages, d.c.page, d.c.W * d.c.page, page_div(d.c.page)};
  p.k = (const uint16_t*)d.c.k; p.k_sp = d.c.k_sp; p.k_sh = d.c.k_sh; p.k_ss = d.c.k_ss;
  p.v = (const uint16_t*)d.c.v; p.v_sp = d.c.v_sp; p.v_sh = d.c.v_sh; p.v_ss = d.c.v_ss;
  p.q = (const uint16_t*)d.q; p.q_sb = d.q_sb; p.q_sh = d.q_sh;
  p.o = (uint16_t*)d.o; p.o_sb = d.o_sb; p.o_sh = d.o_sh;
  p.w = d.weights; p.w_sb = d.w_sb; p.w_sh = d.w_sh;
  p.decay = d.decay;
  p.B = d.c.B; p.H = d.H; p.heads = d.c.heads; p.group = d.H / d.c.heads;
  p.c = d.scale * 1.4426950408889634f;
  p.slots = round_slots(d.c.W, d.c.page);
  const int64_t heads = (int64_t)p.B * p.H;
  if (heads > max_workgroups(256)) return hipErrorNotSupported;
  if (d.weights) {
    p.stat = (float*)d.ws;
    p.scores = p.stat + (2 * heads + 3) / 4 * 4;
  }
  hipLaunchKernelGGL((decode_heads<T, D>), dim3((unsigned)heads), dim3(256), 0, s, p);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess || !d.weights) return e;
  if ((int64_t)p.B * p.heads > 65535) return hipErrorNotSupported;
  const unsigned chunks = (unsigned)std::min<int64_t>((p.slots + 1023) / 1024, 1024);
  hipLaunchKernelGGL(slot_weights, dim3(chunks, (unsigned)(p.B * p.heads)), dim3(256), 0, s, p);
  return hipGetLastError();
}

}  // namespace

size_t paged_attention_workspace(int B, int H, int, int, int W, int page, bool weights) {
  const size_t heads = (size_t)B * H;
  return weights ? ((2 * heads + 3) / 4 * 4 + heads * (size_t)round_slots(W, page)) * sizeof(float) : 0;
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
