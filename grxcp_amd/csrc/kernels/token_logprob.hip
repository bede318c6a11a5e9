// grxDNN log probabilities of given tokens over rows of logits, with entropy and
// the top alternatives, and their gradient in the logits, on gfx950.
//
// New: the reference plans softmax for grxDNN (ref
// docs/designs/grxcp_roadmap.md:864-877) and ships no code.

#include "../launch.h"
#include "device_common.h"
#include "paged_common.h"
#include "row_io.h"

#include <algorithm>

namespace grxk {
namespace {

struct LParams {
  const uint8_t* x;
  int64_t x_rs, rows;
  int vocab, top;
  const int* tokens;
  float* logprob; float* lse; float* entropy;
  float* top_logprob; int* top_index;
};

constexpr int kNT = 256;

// f combined over the workgroup, in every thread.
template <class Op> __device__ __forceinline__ float block_reduce(float v, Op op, float* red) {
  v = wave_reduce(v, op);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  return op(op(red[0], red[1]), op(red[2], red[3]));
}

// A value and its place as one number: larger values first, of equal ones the
// lower place.
__device__ __forceinline__ uint64_t rank_key(float v, int j) {
  return (uint64_t)order_key(__float_as_uint(v)) << 32 | (uint32_t)~j;
}

// One workgroup per row: maximum, sums, then the largest key below the last one
// for every alternative.
template <NormType T>
__global__ __launch_bounds__(kNT) void logprob_rows(LParams p) {
  using IO = Io<T>;
  __shared__ float red[4];
  __shared__ uint64_t keys[4];
  const int tid = threadIdx.x;
  for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
    const uint8_t* x = p.x + row * p.x_rs * (int64_t)(16 / IO::kVec);
    float m = -INFINITY, s = 0.0f, t = 0.0f;
    bool nan = false;
    for (int j = tid; j < p.vocab; j += kNT) {
      const float v = IO::ld(x, j);
      nan |= v != v;
      m = fmaxf(m, v);
    }
    // (not below the lowest finite value: a row of only -inf has sum 0 and lse -inf)
    m = fmaxf(block_reduce(nan ? INFINITY : m, [](float a, float b) { return fmaxf(a, b); }, red), -__FLT_MAX__);
    for (int j = tid; j < p.vocab; j += kNT) {
      const float d = IO::ld(x, j) - m, e = expf(d);
      s += e;
      t += e > 0.0f ? e * d : 0.0f;
    }
    s = block_reduce(s, [](float a, float b) { return a + b; }, red);
    t = block_reduce(t, [](float a, float b) { return a + b; }, red);
    const float ls = logf(s), lse = m + ls;
    if (tid == 0) {
      p.lse[row] = lse;
      if (p.entropy) p.entropy[row] = ls - t / s;
      if (p.tokens) {
        const int k = p.tokens[row];
        p.logprob[row] = (uint32_t)k < (uint32_t)p.vocab ? (IO::ld(x, k) - m) - ls : 0.0f;
      }
    }
    uint64_t last = ~0ull;
    for (int i = 0; i < p.top; ++i) {
      uint64_t best = 0;
      for (int j = tid; j < p.vocab; j += kNT) {
        const uint64_t k = rank_key(IO::ld(x, j), j);
        if (k < last && k > best) best = k;
      }
#pragma unroll
      for (int o = 32; o; o >>= 1) best = max(best, (uint64_t)__shfl_xor((unsigned long long)best, o));
      __syncthreads();
      if ((tid & 63) == 0) keys[tid >> 6] = best;
      __syncthreads();
      last = max(max(keys[0], keys[1]), max(keys[2], keys[3]));
      if (tid == 0) {
        const int j = (int)~(uint32_t)last;
        p.top_index[row * p.top + i] = j;
        p.top_logprob[row * p.top + i] = (IO::ld(x, j) - m) - ls;
      }
    }
  }
}

struct GParams {
  const uint8_t* x;
  uint8_t* dx;
  int64_t x_rs, dx_rs, rows;
  int vocab;
  const int* tokens;
  const float* lse; const float* entropy;
  const float* dlogprob; const float* dentropy;
};

template <NormType T>
__global__ __launch_bounds__(kNT) void logprob_grad(GParams p) {
  using IO = Io<T>;
  for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
    const uint8_t* x = p.x + row * p.x_rs * (int64_t)(16 / IO::kVec);
    uint8_t* dx = p.dx + row * p.dx_rs * (int64_t)(16 / IO::kVec);
    const float lse = p.lse[row];
    const int token = p.tokens ? p.tokens[row] : -1;
    const bool given = (uint32_t)token < (uint32_t)p.vocab;
    const float g = given ? p.dlogprob[row] : 0.0f;
    const float gh = p.entropy ? p.dentropy[row] : 0.0f, h = p.entropy ? p.entropy[row] : 0.0f;
    for (int j = threadIdx.x; j < p.vocab; j += kNT) {
      const float lp = IO::ld(x, j) - lse, e = expf(lp);
      float d = given ? (j == token ? g : 0.0f) - g * e : 0.0f;
      if (p.entropy && e != 0.0f) d -= gh * e * (lp + h);
      IO::st(dx, j, d);
    }
  }
}

template <NormType T>
hipError_t run_forward(const TokenLogProbDesc& d, hipStream_t s) {
  LParams p{};
  p.x = (const uint8_t*)d.x; p.x_rs = d.x_row_stride; p.rows = d.rows; p.vocab = d.vocab; p.top = d.top;
  p.tokens = d.tokens; p.logprob = d.logprob; p.lse = d.lse; p.entropy = d.entropy;
  p.top_logprob = d.top_logprob; p.top_index = d.top_index;
  const unsigned grid = (unsigned)std::min<int64_t>(d.rows, max_workgroups(kNT));
  hipLaunchKernelGGL(logprob_rows<T>, dim3(grid), dim3(kNT), 0, s, p);
  return hipGetLastError();
}

template <NormType T>
hipError_t run_grad(const TokenLogProbGradDesc& d, hipStream_t s) {
  GParams p{};
  p.x = (const uint8_t*)d.x; p.dx = (uint8_t*)d.dx; p.x_rs = d.x_row_stride; p.dx_rs = d.dx_row_stride;
  p.rows = d.rows; p.vocab = d.vocab; p.tokens = d.tokens; p.lse = d.lse; p.entropy = d.entropy;
  p.dlogprob = d.dlogprob; p.dentropy = d.dentropy;
  const unsigned grid = (unsigned)std::min<int64_t>(d.rows, max_workgroups(kNT));
  hipLaunchKernelGGL(logprob_grad<T>, dim3(grid), dim3(kNT), 0, s, p);
  return hipGetLastError();
}

}  // namespace

size_t token_logprob_workspace(NormType, int64_t, int, int) { return 0; }

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
