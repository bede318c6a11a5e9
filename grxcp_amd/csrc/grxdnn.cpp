// libgrxdnn.so -- grxDNN host library for gfx950.
//
// The reference plans grxDNN (ref: src/libs/CMakeLists.txt:12,
// docs/designs/grxcp_architecture.md:594,640, docs/designs/grxcp_roadmap.md:
// 864-877) but ships no code, so this library follows grxBLAS's host
// conventions (ref: src/libs/grxblas/grxblas.cpp): an opaque handle with a
// borrowed stream, every argument validated before any device work, the same
// status values, NOT_SUPPORTED instead of a silent fallback, asynchronous
// launches on the handle's stream.

#include <grx/grxdnn.h>

#include <hip/hip_runtime_api.h>

#include <algorithm>
#include <array>
#include <climits>
#include <cmath>
#include <cstdio>
#include <cstring>
#include <mutex>
#include <new>
#include <utility>

#include "hip_status.h"
#include "launch.h"

struct grxdnnContext {
  hipStream_t stream = nullptr;
  grxCycleSlot* probe = nullptr;
  int probe_capacity = 0;
  std::mutex mutex;
  std::array<signed char, 64> device_ok{};
  grxdnnStatus_t device_status[64];
};

struct grxdnnTensorStruct {
  bool set = false;
  grxDataType_t type = GRX_R_32F;
  int nb = 0;
  int dims[GRXDNN_DIM_MAX] = {0};
  int strides[GRXDNN_DIM_MAX] = {0};
};

struct grxdnnAttentionStruct {
  bool set = false;
  int causal = 0;
  float scale = 1.0f;
};

namespace {

grxdnnStatus_t ensure_device(grxdnnContext& ctx) {
  std::lock_guard<std::mutex> lock(ctx.mutex);
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess || dev < 0) {
    static bool said = false;
    if (!said) {
      said = true;
      std::fprintf(stderr, "grxdnn: no HIP device is available.\n");
    }
    return GRXDNN_STATUS_ARCH_MISMATCH;
  }
  if (dev >= (int)ctx.device_ok.size()) return GRXDNN_STATUS_NOT_SUPPORTED;
  if (ctx.device_ok[dev] == 1) return GRXDNN_STATUS_SUCCESS;
  if (ctx.device_ok[dev] == -1) return ctx.device_status[dev];
  hipDeviceProp_t p;
  grxdnnStatus_t st = GRXDNN_STATUS_SUCCESS;
  if (hipGetDeviceProperties(&p, dev) != hipSuccess) {
    st = GRXDNN_STATUS_INTERNAL_ERROR;
  } else if (std::strncmp(p.gcnArchName, "gfx950", 6) != 0 || p.warpSize != 64) {
    std::fprintf(stderr, "grxdnn: this build carries gfx950 kernels; device %d is %s.\n", dev,
                 p.gcnArchName);
    st = GRXDNN_STATUS_ARCH_MISMATCH;
  }
  ctx.device_ok[dev] = (st == GRXDNN_STATUS_SUCCESS) ? 1 : -1;
  ctx.device_status[dev] = st;
  return st;
}

grxdnnStatus_t from_hip(hipError_t e) {
  switch (grx_from_hip(e)) {
    case grxSuccess:                   return GRXDNN_STATUS_SUCCESS;
    case grxErrorMemoryAllocation:     return GRXDNN_STATUS_ALLOC_FAILED;
    case grxErrorInvalidValue:         return GRXDNN_STATUS_INVALID_VALUE;
    case grxErrorInvalidDevicePointer: return GRXDNN_STATUS_INVALID_VALUE;
    case grxErrorNotSupported:         return GRXDNN_STATUS_NOT_SUPPORTED;
    case grxErrorInvalidKernelImage:   return GRXDNN_STATUS_ARCH_MISMATCH;
    default:                           return GRXDNN_STATUS_EXECUTION_FAILED;
  }
}

bool known_type(grxDataType_t t) {
  return t == GRX_R_32F || t == GRX_R_16F || t == GRX_R_8I || t == GRX_R_32I || t == GRX_R_16BF;
}

bool same_shape(const grxdnnTensorStruct& a, const grxdnnTensorStruct& b) {
  if (a.nb != b.nb) return false;
  for (int i = 0; i < a.nb; ++i)
    if (a.dims[i] != b.dims[i]) return false;
  return true;
}

// Rows of a [..., hidden] tensor: all leading dimensions must collapse into
// one row index with a single pitch. Returns false if they do not. What a
// dimension of extent 1 has for a stride does not matter.
bool row_layout(const grxdnnTensorStruct& t, int64_t* rows, int64_t* pitch) {
  const int hidden = t.dims[t.nb - 1];
  *rows = 1;
  *pitch = t.nb == 1 ? hidden : t.strides[t.nb - 2];
  int64_t next = -1;               // what the next outer stride has to be, from the first extent above 1 on
  for (int i = t.nb - 2; i >= 0; --i) {
    *rows *= t.dims[i];
    if (t.dims[i] == 1) continue;
    if (next < 0) *pitch = t.strides[i];
    else if (t.strides[i] != next) return false;
    next = (int64_t)t.strides[i] * t.dims[i];
  }
  return *pitch >= hidden || *rows <= 1;
}

bool aligned16(const void* p) { return ((uintptr_t)p % 16) == 0; }

// No two elements of an output share an address: taken in increasing stride
// order (dimensions of extent 1 aside), each stride covers the extent of the
// dimensions below it. An input may overlap itself (a broadcast); an output
// that did would be written by several threads.
bool no_overlap(const grxdnnTensorStruct& t) {
  int idx[GRXDNN_DIM_MAX];
  int n = 0;
  for (int i = 0; i < t.nb; ++i)
    if (t.dims[i] > 1) idx[n++] = i;
  for (int a = 1; a < n; ++a)
    for (int b = a; b > 0 && t.strides[idx[b]] < t.strides[idx[b - 1]]; --b) {
      const int x = idx[b];
      idx[b] = idx[b - 1];
      idx[b - 1] = x;
    }
  int64_t extent = 1;
  for (int j = 0; j < n; ++j) {
    const int i = idx[j];
    if ((int64_t)t.strides[i] < extent) return false;
    extent = (int64_t)t.strides[i] * t.dims[i];
  }
  return true;
}

// Byte interval [lo, hi) covered by a tensor at p (strides are non-negative).
struct Span { uintptr_t lo, hi; };
Span span_of(const grxdnnTensorStruct& t, const void* p, size_t elem) {
  int64_t last = 0;
  for (int i = 0; i < t.nb; ++i)
    if (t.dims[i] > 0) last += (int64_t)t.strides[i] * (t.dims[i] - 1);
  const uintptr_t lo = (uintptr_t)p;
  return {lo, lo + (uintptr_t)((last + 1) * (int64_t)elem)};
}
bool intersect(Span a, Span b) { return a.lo < b.hi && b.lo < a.hi; }

bool same_strides(const grxdnnTensorStruct& a, const grxdnnTensorStruct& b) {
  for (int i = 0; i < a.nb; ++i)
    if (a.strides[i] != b.strides[i]) return false;
  return true;
}

// Whether delta = sum_i strides[i] * d_i has a solution with |d_i| <
// extents[i], for dimensions taken in decreasing stride order from `from`;
// reach[i] is the largest |sum| the dimensions after i can make. Returns
// true ("may share an element") when the search would take too many steps.
bool offset_reachable(const int64_t* strides, const int64_t* extents, const int64_t* reach,
                      int n, int from, int64_t delta, int* budget) {
  if (from == n) return delta == 0;
  const int64_t s = strides[from], r = reach[from], e = extents[from] - 1;
  // d with |delta - s*d| <= r: d in [ceil((delta-r)/s), floor((delta+r)/s)]
  auto floor_div = [](int64_t a, int64_t b) { return a >= 0 ? a / b : -((-a + b - 1) / b); };
  int64_t lo = -floor_div(-(delta - r), s), hi = floor_div(delta + r, s);
  if (lo < -e) lo = -e;
  if (hi > e) hi = e;
  for (int64_t d = lo; d <= hi; ++d) {
    if (--*budget < 0) return true;
    if (offset_reachable(strides, extents, reach, n, from + 1, delta - s * d, budget)) return true;
  }
  return false;
}

// Two views of one shape and the same strides (bases a and b, elements of
// `elem` bytes) share an element's address. An exact test of the element
// offsets, so that e.g. O written over the Q slot of a packed [B,S,3,H,D]
// QKV buffer is told apart from O overlapping K or V. Views whose bases do
// not differ by whole elements are taken to overlap when their spans do.
bool views_share_element(const grxdnnTensorStruct& t, const void* a, const void* b, size_t elem) {
  const int64_t diff = (int64_t)((intptr_t)b - (intptr_t)a);
  if (diff % (int64_t)elem != 0) return intersect(span_of(t, a, elem), span_of(t, b, elem));
  int64_t strides[GRXDNN_DIM_MAX], extents[GRXDNN_DIM_MAX], reach[GRXDNN_DIM_MAX];
  int n = 0;
  for (int i = 0; i < t.nb; ++i) {
    if (t.dims[i] <= 0) return false;                      // an empty view
    if (t.dims[i] == 1 || t.strides[i] == 0) continue;     // contributes no offset
    strides[n] = t.strides[i];
    extents[n] = t.dims[i];
    ++n;
  }
  for (int x = 1; x < n; ++x)                              // decreasing stride
    for (int y = x; y > 0 && strides[y] > strides[y - 1]; --y) {
      std::swap(strides[y], strides[y - 1]);
      std::swap(extents[y], extents[y - 1]);
    }
  int64_t acc = 0;
  for (int i = n - 1; i >= 0; --i) {
    reach[i] = acc;
    acc += strides[i] * (extents[i] - 1);
  }
  int budget = 4096;
  return offset_reachable(strides, extents, reach, n, 0, diff / (int64_t)elem, &budget);
}

// O may share no element with x: the exact test where the two views have the
// same strides, the span test otherwise.
bool may_alias(const grxdnnTensorStruct& od, const void* o, const grxdnnTensorStruct& xd,
               const void* x) {
  if (same_strides(od, xd)) return views_share_element(od, o, x, 2);
  return intersect(span_of(od, o, 2), span_of(xd, x, 2));
}

grxdnnStatus_t norm_common(grxdnnHandle_t handle, grxdnnTensorDescriptor_t xDesc, const void* x,
                           grxdnnTensorDescriptor_t wDesc, const void* gamma, const void* beta,
                           bool layer, float eps, grxdnnTensorDescriptor_t yDesc, void* y) {
  if (!handle) return GRXDNN_STATUS_NOT_INITIALIZED;
  if (!xDesc || !wDesc || !yDesc) return GRXDNN_STATUS_INVALID_VALUE;
  if (!xDesc->set || !wDesc->set || !yDesc->set) return GRXDNN_STATUS_INVALID_VALUE;
  if (!same_shape(*xDesc, *yDesc)) return GRXDNN_STATUS_INVALID_VALUE;
  const int hidden = xDesc->dims[xDesc->nb - 1];
  if (wDesc->nb != 1 || wDesc->dims[0] != hidden) return GRXDNN_STATUS_INVALID_VALUE;
  if (!std::isfinite(eps) || eps < 0.0f) return GRXDNN_STATUS_INVALID_VALUE;
  if (xDesc->type != yDesc->type || xDesc->type != wDesc->type) return GRXDNN_STATUS_NOT_SUPPORTED;
  grxk::NormType nt;
  switch (xDesc->type) {
    case GRX_R_16BF: nt = grxk::NormType::BF16; break;
    case GRX_R_16F:  nt = grxk::NormType::F16; break;
    case GRX_R_32F:  nt = grxk::NormType::F32; break;
    default: return GRXDNN_STATUS_NOT_SUPPORTED;
  }
  int64_t rows = 0, xp = 0, yp = 0, yrows = 0;
  for (int i = 0; i < xDesc->nb - 1; ++i)
    if (xDesc->dims[i] == 0) return GRXDNN_STATUS_SUCCESS;  // no rows: nothing to do
  if (hidden <= 0) return GRXDNN_STATUS_INVALID_VALUE;
  if (hidden > 65536) return GRXDNN_STATUS_NOT_SUPPORTED;
  if (xDesc->strides[xDesc->nb - 1] != 1 || yDesc->strides[yDesc->nb - 1] != 1 ||
      wDesc->strides[0] != 1)
    return GRXDNN_STATUS_NOT_SUPPORTED;
  if (!row_layout(*xDesc, &rows, &xp) || !row_layout(*yDesc, &yrows, &yp))
    return GRXDNN_STATUS_NOT_SUPPORTED;
  if (!x || !gamma || !y || (layer && !beta)) return GRXDNN_STATUS_INVALID_VALUE;

  const grxdnnStatus_t s = ensure_device(*handle);
  if (s != GRXDNN_STATUS_SUCCESS) return s;

  grxk::NormDesc d{};
  d.rows = rows;
  d.hidden = hidden;
  d.x_row_stride = xp;
  d.y_row_stride = yp;
  d.x = x; d.gamma = gamma; d.beta = beta; d.y = y;
  d.eps = eps;
  const hipError_t e = layer ? grxk::launch_layernorm(nt, d, handle->stream)
                             : grxk::launch_rmsnorm(nt, d, handle->stream);
  return from_hip(e);
}

// Softmax / GELU: x and y of one type and shape, rows flattening to one
// stride each, innermost stride 1.
grxdnnStatus_t row_common(grxdnnHandle_t handle, grxdnnTensorDescriptor_t xDesc, const void* x,
                          grxdnnTensorDescriptor_t yDesc, void* y, grxk::NormType* nt,
                          grxk::RowDesc* d, bool* empty) {
  *empty = false;
  if (!handle) return GRXDNN_STATUS_NOT_INITIALIZED;
  if (!xDesc || !yDesc || !xDesc->set || !yDesc->set) return GRXDNN_STATUS_INVALID_VALUE;
  if (!same_shape(*xDesc, *yDesc)) return GRXDNN_STATUS_INVALID_VALUE;
  if (xDesc->type != yDesc->type) return GRXDNN_STATUS_NOT_SUPPORTED;
  switch (xDesc->type) {
    case GRX_R_16BF: *nt = grxk::NormType::BF16; break;
    case GRX_R_16F:  *nt = grxk::NormType::F16; break;
    case GRX_R_32F:  *nt = grxk::NormType::F32; break;
    default: return GRXDNN_STATUS_NOT_SUPPORTED;
  }
  for (int i = 0; i < xDesc->nb - 1; ++i)
    if (xDesc->dims[i] == 0) {  // no rows: nothing to do
      *empty = true;
      return GRXDNN_STATUS_SUCCESS;
    }
  const int hidden = xDesc->dims[xDesc->nb - 1];
  if (hidden <= 0) return GRXDNN_STATUS_INVALID_VALUE;
  if (hidden > (1 << 24)) return GRXDNN_STATUS_NOT_SUPPORTED;
  if (xDesc->strides[xDesc->nb - 1] != 1 || yDesc->strides[yDesc->nb - 1] != 1)
    return GRXDNN_STATUS_NOT_SUPPORTED;
  int64_t rows = 0, yrows = 0, xp = 0, yp = 0;
  if (!row_layout(*xDesc, &rows, &xp) || !row_layout(*yDesc, &yrows, &yp))
    return GRXDNN_STATUS_NOT_SUPPORTED;
  if (!x || !y) return GRXDNN_STATUS_INVALID_VALUE;
  const grxdnnStatus_t s = ensure_device(*handle);
  if (s != GRXDNN_STATUS_SUCCESS) return s;
  d->rows = rows;
  d->hidden = hidden;
  d->x_row_stride = xp;
  d->y_row_stride = yp;
  d->x = x;
  d->y = y;
  return GRXDNN_STATUS_SUCCESS;
}

bool half_type(grxDataType_t t) { return t == GRX_R_16BF || t == GRX_R_16F; }

// 16-byte vector access along the last dimension: contiguous, rows on 16 bytes.
bool half_rows(const grxdnnTensorStruct& t) {
  if (t.strides[t.nb - 1] != 1) return false;
  for (int i = 0; i < t.nb - 1; ++i)
    if (t.dims[i] > 1 && t.strides[i] % 8 != 0) return false;
  return true;
}

// Slots that a sequence may have room for: the kernels count them in 32 bits, up to a
// tile's or a workgroup's worth past the last.
constexpr int kMaxRoom = INT_MAX - 4095;

// A table of pages: [B, W] ints, rows of any pitch.
bool table_shape(const grxdnnTensorStruct& t) {
  return t.nb == 2 && t.type == GRX_R_32I && t.dims[1] >= 1 && (t.dims[1] == 1 || t.strides[1] == 1);
}

// fp32 [B, heads, S] of S >= slots with contiguous slots.
bool weights_shape(const grxdnnTensorStruct& t, int B, int heads, int64_t slots) {
  return t.nb == 3 && t.type == GRX_R_32F && t.dims[0] == B && t.dims[1] == heads && t.dims[2] >= slots &&
         (t.dims[2] <= 1 || t.strides[2] == 1);
}

// The pools and the table of a paged call, but for their pointers.
grxdnnStatus_t paged_cache(grxdnnTensorDescriptor_t kDesc, grxdnnTensorDescriptor_t vDesc,
                           grxdnnTensorDescriptor_t tableDesc, bool written, grxk::PagedCache* c) {
  if (!kDesc || !vDesc || !tableDesc || !kDesc->set || !vDesc->set || !tableDesc->set)
    return GRXDNN_STATUS_INVALID_VALUE;
  if (kDesc->nb != 4 || !same_shape(*kDesc, *vDesc) || !table_shape(*tableDesc))
    return GRXDNN_STATUS_INVALID_VALUE;
  for (int i = 0; i < 4; ++i)
    if (kDesc->dims[i] < 1) return GRXDNN_STATUS_INVALID_VALUE;
  if (!half_type(kDesc->type) || vDesc->type != kDesc->type) return GRXDNN_STATUS_NOT_SUPPORTED;
  c->pages = kDesc->dims[0];
  c->heads = kDesc->dims[1];
  c->page = kDesc->dims[2];
  c->D = kDesc->dims[3];
  c->B = tableDesc->dims[0];
  c->W = tableDesc->dims[1];
  c->table_rs = tableDesc->strides[0];
  if (c->D != 64 && c->D != 128) return GRXDNN_STATUS_NOT_SUPPORTED;
  if ((int64_t)c->W * c->page > kMaxRoom) return GRXDNN_STATUS_NOT_SUPPORTED;
  // (sequence, head) pairs are counted in 32 bits
  if ((int64_t)c->B * c->heads > INT_MAX / 4) return GRXDNN_STATUS_NOT_SUPPORTED;
  if (!half_rows(*kDesc) || !half_rows(*vDesc)) return GRXDNN_STATUS_NOT_SUPPORTED;
  if (written && (!no_overlap(*kDesc) || !no_overlap(*vDesc))) return GRXDNN_STATUS_INVALID_VALUE;
  c->k_sp = kDesc->strides[0]; c->k_sh = kDesc->strides[1]; c->k_ss = kDesc->strides[2];
  c->v_sp = vDesc->strides[0]; c->v_sh = vDesc->strides[1]; c->v_ss = vDesc->strides[2];
  return GRXDNN_STATUS_SUCCESS;
}

Span bytes_at(const void* p, int64_t n) { return {(uintptr_t)p, (uintptr_t)p + (uintptr_t)n}; }

// Logits of softmax's layout: rows, their pitch and the element type.
grxdnnStatus_t logit_rows(const grxdnnTensorStruct& x, grxk::NormType* nt, int64_t* rows, int64_t* pitch) {
  switch (x.type) {
    case GRX_R_16BF: *nt = grxk::NormType::BF16; break;
    case GRX_R_16F:  *nt = grxk::NormType::F16; break;
    case GRX_R_32F:  *nt = grxk::NormType::F32; break;
    default: return GRXDNN_STATUS_NOT_SUPPORTED;
  }
  const int vocab = x.dims[x.nb - 1];
  *rows = 1;
  for (int i = 0; i < x.nb - 1; ++i)
    if (x.dims[i] == 0) *rows = 0;
  if (vocab <= 0) return *rows ? GRXDNN_STATUS_INVALID_VALUE : GRXDNN_STATUS_SUCCESS;
  if (vocab > (1 << 24)) return GRXDNN_STATUS_NOT_SUPPORTED;
  if (x.strides[x.nb - 1] != 1) return GRXDNN_STATUS_NOT_SUPPORTED;
  if (*rows && !row_layout(x, rows, pitch)) return GRXDNN_STATUS_NOT_SUPPORTED;
  return GRXDNN_STATUS_SUCCESS;
}

size_t element_size(grxk::NormType t) { return t == grxk::NormType::F32 ? 4 : 2; }

}  // namespace

// The C API is the only thing these libraries export (built with
// -fvisibility=hidden).
#pragma GCC visibility push(default)
extern "C" {

const char* grxdnnGetStatusString(grxdnnStatus_t s) {
  switch (s) {
    case GRXDNN_STATUS_SUCCESS:          return "success";
    case GRXDNN_STATUS_NOT_INITIALIZED:  return "library not initialized";
    case GRXDNN_STATUS_ALLOC_FAILED:     return "allocation failed";
    case GRXDNN_STATUS_INVALID_VALUE:    return "invalid argument";
    case GRXDNN_STATUS_ARCH_MISMATCH:    return "device lacks a required capability";
    case GRXDNN_STATUS_EXECUTION_FAILED: return "kernel execution failed";
    case GRXDNN_STATUS_NOT_SUPPORTED:    return "not supported";
    case GRXDNN_STATUS_INTERNAL_ERROR:   return "internal error";
  }
  return "unknown status";
}

grxdnnStatus_t grxdnnCreate(grxdnnHandle_t* handle) {
  if (!handle) return GRXDNN_STATUS_INVALID_VALUE;
  *handle = new (std::nothrow) grxdnnContext();
  return *handle ? GRXDNN_STATUS_SUCCESS : GRXDNN_STATUS_ALLOC_FAILED;
}

grxdnnStatus_t grxdnnDestroy(grxdnnHandle_t handle) {
  if (!handle) return GRXDNN_STATUS_NOT_INITIALIZED;
  delete handle;
  return GRXDNN_STATUS_SUCCESS;
}

grxdnnStatus_t grxdnnSetStream(grxdnnHandle_t handle, grxStream_t stream) {
  if (!handle) return GRXDNN_STATUS_NOT_INITIALIZED;
  handle->stream = reinterpret_cast<hipStream_t>(stream);
  return GRXDNN_STATUS_SUCCESS;
}

grxdnnStatus_t grxdnnGetStream(grxdnnHandle_t handle, grxStream_t* stream) {
  if (!handle || !stream) return GRXDNN_STATUS_INVALID_VALUE;
  *stream = reinterpret_cast<grxStream_t>(handle->stream);
  return GRXDNN_STATUS_SUCCESS;
}

grxdnnStatus_t grxdnnCreateTensorDescriptor(grxdnnTensorDescriptor_t* desc) {
  if (!desc) return GRXDNN_STATUS_INVALID_VALUE;
  *desc = new (std::nothrow) grxdnnTensorStruct();
  return *desc ? GRXDNN_STATUS_SUCCESS : GRXDNN_STATUS_ALLOC_FAILED;
}

grxdnnStatus_t grxdnnDestroyTensorDescriptor(grxdnnTensorDescriptor_t desc) {
  if (!desc) return GRXDNN_STATUS_INVALID_VALUE;
  delete desc;
  return GRXDNN_STATUS_SUCCESS;
}

grxdnnStatus_t grxdnnSetTensorNdDescriptor(grxdnnTensorDescriptor_t desc, grxDataType_t dataType,
                                           int nbDims, const int dims[], const int strides[]) {
  if (!desc || !dims) return GRXDNN_STATUS_INVALID_VALUE;
  if (nbDims < 1 || nbDims > GRXDNN_DIM_MAX) return GRXDNN_STATUS_INVALID_VALUE;
  if (!known_type(dataType)) return GRXDNN_STATUS_INVALID_VALUE;
  for (int i = 0; i < nbDims; ++i) {
    if (dims[i] < 0) return GRXDNN_STATUS_INVALID_VALUE;
    if (strides && strides[i] < 0) return GRXDNN_STATUS_INVALID_VALUE;
  }
  grxdnnTensorStruct t;
  t.set = true;
  t.type = dataType;
  t.nb = nbDims;
  int64_t packed = 1;
  for (int i = nbDims - 1; i >= 0; --i) {
    t.dims[i] = dims[i];
    if (strides) {
      t.strides[i] = strides[i];
    } else {
      if (packed > 0x7fffffff) return GRXDNN_STATUS_INVALID_VALUE;
      t.strides[i] = (int)packed;
    }
    packed *= (dims[i] > 0 ? dims[i] : 1);
  }
  *desc = t;
  return GRXDNN_STATUS_SUCCESS;
}

grxdnnStatus_t grxdnnGetTensorNdDescriptor(grxdnnTensorDescriptor_t desc, int nbDimsRequested,
                                           grxDataType_t* dataType, int* nbDims, int dims[],
                                           int strides[]) {
  if (!desc || !desc->set) return GRXDNN_STATUS_INVALID_VALUE;
  if (nbDimsRequested < 0) return GRXDNN_STATUS_INVALID_VALUE;
  if (dataType) *dataType = desc->type;
  if (nbDims) *nbDims = desc->nb;
  const int n = nbDimsRequested < desc->nb ? nbDimsRequested : desc->nb;
  for (int i = 0; i < n; ++i) {
    if (dims) dims[i] = desc->dims[i];
    if (strides) strides[i] = desc->strides[i];
  }
  return GRXDNN_STATUS_SUCCESS;
}

grxdnnStatus_t grxdnnRMSNormForward(grxdnnHandle_t handle, grxdnnTensorDescriptor_t xDesc,
                                    const void* x, grxdnnTensorDescriptor_t wDesc,
                                    const void* gamma, float eps, grxdnnTensorDescriptor_t yDesc,
                                    void* y) {
  return norm_common(handle, xDesc, x, wDesc, gamma, nullptr, false, eps, yDesc, y);
}

grxdnnStatus_t grxdnnLayerNormForward(grxdnnHandle_t handle, grxdnnTensorDescriptor_t xDesc,
                                      const void* x, grxdnnTensorDescriptor_t wDesc,
                                      const void* gamma, const void* beta, float eps,
                                      grxdnnTensorDescriptor_t yDesc, void* y) {
  return norm_common(handle, xDesc, x, wDesc, gamma, beta, true, eps, yDesc, y);
}

grxdnnStatus_t grxdnnSoftmaxForward(grxdnnHandle_t handle, grxdnnTensorDescriptor_t xDesc,
                                    const void* x, grxdnnTensorDescriptor_t yDesc, void* y) {
  grxk::NormType nt{};
  grxk::RowDesc d{};
  bool empty = false;
  const grxdnnStatus_t s = row_common(handle, xDesc, x, yDesc, y, &nt, &d, &empty);
  if (s != GRXDNN_STATUS_SUCCESS || empty) return s;
  return from_hip(grxk::launch_softmax(nt, d, handle->stream));
}

grxdnnStatus_t grxdnnGeluForward(grxdnnHandle_t handle, grxdnnGeluMode_t mode,
                                 grxdnnTensorDescriptor_t xDesc, const void* x,
                                 grxdnnTensorDescriptor_t yDesc, void* y) {
  if (!handle) return GRXDNN_STATUS_NOT_INITIALIZED;
  if (mode != GRXDNN_GELU_ERF && mode != GRXDNN_GELU_TANH) return GRXDNN_STATUS_INVALID_VALUE;
  grxk::NormType nt{};
  grxk::RowDesc d{};
  bool empty = false;
  const grxdnnStatus_t s = row_common(handle, xDesc, x, yDesc, y, &nt, &d, &empty);
  if (s != GRXDNN_STATUS_SUCCESS || empty) return s;
  return from_hip(grxk::launch_gelu(nt, mode == GRXDNN_GELU_TANH, d, handle->stream));
}

grxdnnStatus_t grxdnnCreateAttentionDescriptor(grxdnnAttentionDescriptor_t* d) {
  if (!d) return GRXDNN_STATUS_INVALID_VALUE;
  *d = new (std::nothrow) grxdnnAttentionStruct();
  return *d ? GRXDNN_STATUS_SUCCESS : GRXDNN_STATUS_ALLOC_FAILED;
}

grxdnnStatus_t grxdnnDestroyAttentionDescriptor(grxdnnAttentionDescriptor_t d) {
  if (!d) return GRXDNN_STATUS_INVALID_VALUE;
  delete d;
  return GRXDNN_STATUS_SUCCESS;
}

grxdnnStatus_t grxdnnSetAttentionDescriptor(grxdnnAttentionDescriptor_t d, int causal,
                                            float softmaxScale) {
  if (!d) return GRXDNN_STATUS_INVALID_VALUE;
  if (causal != 0 && causal != 1) return GRXDNN_STATUS_INVALID_VALUE;
  if (!std::isfinite(softmaxScale) || softmaxScale <= 0.0f) return GRXDNN_STATUS_INVALID_VALUE;
  d->set = true;
  d->causal = causal;
  d->scale = softmaxScale;
  return GRXDNN_STATUS_SUCCESS;
}

grxdnnStatus_t grxdnnGetAttentionDescriptor(grxdnnAttentionDescriptor_t d, int* causal,
                                            float* softmaxScale) {
  if (!d || !d->set) return GRXDNN_STATUS_INVALID_VALUE;
  if (causal) *causal = d->causal;
  if (softmaxScale) *softmaxScale = d->scale;
  return GRXDNN_STATUS_SUCCESS;
}

grxdnnStatus_t grxdnnAttentionForward(grxdnnHandle_t handle, grxdnnAttentionDescriptor_t attnDesc,
                                      grxdnnTensorDescriptor_t qDesc, const void* q,
                                      grxdnnTensorDescriptor_t kDesc, const void* k,
                                      grxdnnTensorDescriptor_t vDesc, const void* v,
                                      grxdnnTensorDescriptor_t oDesc, void* o) {
  if (!handle) return GRXDNN_STATUS_NOT_INITIALIZED;
  if (!attnDesc || !qDesc || !kDesc || !vDesc || !oDesc) return GRXDNN_STATUS_INVALID_VALUE;
  if (!attnDesc->set || !qDesc->set || !kDesc->set || !vDesc->set || !oDesc->set)
    return GRXDNN_STATUS_INVALID_VALUE;
  if (qDesc->nb != 4 || !same_shape(*qDesc, *kDesc) || !same_shape(*qDesc, *vDesc) ||
      !same_shape(*qDesc, *oDesc))
    return GRXDNN_STATUS_INVALID_VALUE;
  const grxDataType_t t = qDesc->type;
  if (kDesc->type != t || vDesc->type != t || oDesc->type != t) return GRXDNN_STATUS_NOT_SUPPORTED;
  if (t != GRX_R_16BF && t != GRX_R_16F) return GRXDNN_STATUS_NOT_SUPPORTED;
  const int B = qDesc->dims[0], H = qDesc->dims[1], S = qDesc->dims[2], D = qDesc->dims[3];
  if (D != 64 && D != 128) return GRXDNN_STATUS_NOT_SUPPORTED;
  if ((int64_t)B * H * S == 0) return GRXDNN_STATUS_SUCCESS;
  const grxdnnTensorStruct* all[4] = {qDesc, kDesc, vDesc, oDesc};
  for (const grxdnnTensorStruct* d : all) {
    // 16-byte vector access along the head dimension needs a contiguous head
    // dimension and 16-byte aligned rows.
    if (d->strides[3] != 1) return GRXDNN_STATUS_NOT_SUPPORTED;
    for (int i = 0; i < 3; ++i)
      if (d->strides[i] % 8 != 0) return GRXDNN_STATUS_NOT_SUPPORTED;
  }
  if (!no_overlap(*oDesc)) return GRXDNN_STATUS_INVALID_VALUE;
  if (!q || !k || !v || !o) return GRXDNN_STATUS_INVALID_VALUE;
  // A workgroup writes its O rows while workgroups of other query tiles of
  // the same head still read K and V, so O may not share an element with
  // them. O == Q with the same layout is safe (a workgroup reads only its own
  // Q rows, before it writes them); any other overlap with Q is refused too.
  // Views with O's strides are compared element by element (O over the Q
  // slot of a packed QKV buffer is accepted), others by their byte spans.
  if (may_alias(*oDesc, o, *kDesc, k) || may_alias(*oDesc, o, *vDesc, v))
    return GRXDNN_STATUS_INVALID_VALUE;
  if (may_alias(*oDesc, o, *qDesc, q) && !(o == q && same_strides(*oDesc, *qDesc)))
    return GRXDNN_STATUS_INVALID_VALUE;
  if (!aligned16(q) || !aligned16(k) || !aligned16(v) || !aligned16(o))
    return GRXDNN_STATUS_NOT_SUPPORTED;

  const grxdnnStatus_t s = ensure_device(*handle);
  if (s != GRXDNN_STATUS_SUCCESS) return s;

  grxk::AttnDesc d{};
  d.B = B; d.H = H; d.S = S; d.D = D;
  d.causal = attnDesc->causal != 0;
  d.scale = attnDesc->scale;
  d.q = q; d.q_sb = qDesc->strides[0]; d.q_sh = qDesc->strides[1]; d.q_ss = qDesc->strides[2];
  d.k = k; d.k_sb = kDesc->strides[0]; d.k_sh = kDesc->strides[1]; d.k_ss = kDesc->strides[2];
  d.v = v; d.v_sb = vDesc->strides[0]; d.v_sh = vDesc->strides[1]; d.v_ss = vDesc->strides[2];
  d.o = o; d.o_sb = oDesc->strides[0]; d.o_sh = oDesc->strides[1]; d.o_ss = oDesc->strides[2];
  {
    std::lock_guard<std::mutex> lock(handle->mutex);
    if (handle->probe) {
      if (handle->probe_capacity < grxk::attention_probe_slots(B, H, S))
        return GRXDNN_STATUS_INVALID_VALUE;
      d.probe = handle->probe;
    }
  }
  return from_hip(grxk::launch_attention(
      t == GRX_R_16BF ? grxk::AttnType::BF16 : grxk::AttnType::F16, d, handle->stream));
}

grxdnnStatus_t grxdnnSetCycleProbe(grxdnnHandle_t handle, grxCycleSlot* slots, int capacity) {
  if (!handle) return GRXDNN_STATUS_NOT_INITIALIZED;
  if (slots && capacity <= 0) return GRXDNN_STATUS_INVALID_VALUE;
  std::lock_guard<std::mutex> lock(handle->mutex);
  handle->probe = slots;
  handle->probe_capacity = slots ? capacity : 0;
  return GRXDNN_STATUS_SUCCESS;
}

int grxdnnAttentionCycleSlotsNeeded(grxdnnHandle_t handle, int batch, int heads, int seqLen) {
  (void)handle;
  if (batch <= 0 || heads <= 0 || seqLen <= 0) return 0;
  const int64_t s = grxk::attention_probe_slots(batch, heads, seqLen);
  return s > INT_MAX ? INT_MAX : (int)s;
}

grxdnnStatus_t grxdnnPagedCacheAppend(grxdnnHandle_t handle, grxdnnTensorDescriptor_t kDesc, const void* k,
                                      grxdnnTensorDescriptor_t vDesc, const void* v,
                                      grxdnnTensorDescriptor_t kCacheDesc, void* kCache,
                                      grxdnnTensorDescriptor_t vCacheDesc, void* vCache,
                                      grxdnnTensorDescriptor_t tableDesc, const int* table,
                                      const int* lengths, const int* counts) {
  if (!handle) return GRXDNN_STATUS_NOT_INITIALIZED;
  if (!kDesc || !vDesc || !kDesc->set || !vDesc->set) return GRXDNN_STATUS_INVALID_VALUE;
  grxk::PagedAppendDesc d{};
  grxdnnStatus_t s = paged_cache(kCacheDesc, vCacheDesc, tableDesc, true, &d.c);
  if (s != GRXDNN_STATUS_SUCCESS) return s;
  if (kDesc->nb != 4 || !same_shape(*kDesc, *vDesc) || kDesc->dims[0] != d.c.B ||
      kDesc->dims[1] != d.c.heads || kDesc->dims[3] != d.c.D)
    return GRXDNN_STATUS_INVALID_VALUE;
  if (kDesc->type != kCacheDesc->type || vDesc->type != kCacheDesc->type) return GRXDNN_STATUS_NOT_SUPPORTED;
  d.T = kDesc->dims[2];
  if (d.c.B == 0 || d.T == 0) return GRXDNN_STATUS_SUCCESS;
  if (!half_rows(*kDesc) || !half_rows(*vDesc)) return GRXDNN_STATUS_NOT_SUPPORTED;
  if (!k || !v || !kCache || !vCache || !table || !lengths) return GRXDNN_STATUS_INVALID_VALUE;
  if (may_alias(*kCacheDesc, kCache, *vCacheDesc, vCache)) return GRXDNN_STATUS_INVALID_VALUE;
  for (const auto& [cd, cp] : {std::pair{kCacheDesc, kCache}, std::pair{vCacheDesc, vCache}}) {
    const Span c = span_of(*cd, cp, 2);
    if (intersect(c, span_of(*kDesc, k, 2)) || intersect(c, span_of(*vDesc, v, 2)) ||
        intersect(c, span_of(*tableDesc, table, 4)) || intersect(c, bytes_at(lengths, 4ll * d.c.B)) ||
        (counts && intersect(c, bytes_at(counts, 4ll * d.c.B))))
      return GRXDNN_STATUS_INVALID_VALUE;
  }
  if (!aligned16(k) || !aligned16(v) || !aligned16(kCache) || !aligned16(vCache))
    return GRXDNN_STATUS_NOT_SUPPORTED;
  s = ensure_device(*handle);
  if (s != GRXDNN_STATUS_SUCCESS) return s;
  d.c.k = kCache; d.c.v = vCache; d.c.table = table; d.c.lengths = lengths;
  d.k = k; d.k_sb = kDesc->strides[0]; d.k_sh = kDesc->strides[1]; d.k_st = kDesc->strides[2];
  d.v = v; d.v_sb = vDesc->strides[0]; d.v_sh = vDesc->strides[1]; d.v_st = vDesc->strides[2];
  d.counts = counts;
  return from_hip(grxk::launch_paged_append(d, handle->stream));
}

grxdnnStatus_t grxdnnPagedAttentionGetWorkspaceSize(grxdnnHandle_t handle, grxdnnTensorDescriptor_t qDesc,
                                                    grxdnnTensorDescriptor_t kCacheDesc,
                                                    grxdnnTensorDescriptor_t tableDesc,
                                                    grxdnnTensorDescriptor_t weightsDesc, size_t* bytes) {
  if (!handle) return GRXDNN_STATUS_NOT_INITIALIZED;
  if (!qDesc || !qDesc->set || !bytes) return GRXDNN_STATUS_INVALID_VALUE;
  grxk::PagedCache c{};
  const grxdnnStatus_t s = paged_cache(kCacheDesc, kCacheDesc, tableDesc, false, &c);
  if (s != GRXDNN_STATUS_SUCCESS) return s;
  if (weightsDesc && !weightsDesc->set) return GRXDNN_STATUS_INVALID_VALUE;
  if (qDesc->nb != 4 || qDesc->dims[0] != c.B || qDesc->dims[1] < 1 || qDesc->dims[1] % c.heads != 0 ||
      qDesc->dims[3] != c.D)
    return GRXDNN_STATUS_INVALID_VALUE;
  *bytes = c.B == 0 ? 0 : grxk::paged_attention_workspace(c, qDesc->dims[1], weightsDesc != nullptr);
  return GRXDNN_STATUS_SUCCESS;
}

grxdnnStatus_t grxdnnPagedAttentionForward(grxdnnHandle_t handle, grxdnnAttentionDescriptor_t attnDesc,
                                           grxdnnTensorDescriptor_t qDesc, const void* q,
                                           grxdnnTensorDescriptor_t kCacheDesc, const void* kCache,
                                           grxdnnTensorDescriptor_t vCacheDesc, const void* vCache,
                                           grxdnnTensorDescriptor_t tableDesc, const int* table,
                                           const int* lengths, float weightDecay,
                                           grxdnnTensorDescriptor_t weightsDesc, float* weights,
                                           grxdnnTensorDescriptor_t oDesc, void* o, void* workspace,
                                           size_t workspaceBytes) {
  if (!handle) return GRXDNN_STATUS_NOT_INITIALIZED;
  if (!attnDesc || !qDesc || !oDesc || !attnDesc->set || !qDesc->set || !oDesc->set)
    return GRXDNN_STATUS_INVALID_VALUE;
  if ((weightsDesc != nullptr) != (weights != nullptr) || (weightsDesc && !weightsDesc->set))
    return GRXDNN_STATUS_INVALID_VALUE;
  grxk::PagedAttnDesc d{};
  grxdnnStatus_t s = paged_cache(kCacheDesc, vCacheDesc, tableDesc, false, &d.c);
  if (s != GRXDNN_STATUS_SUCCESS) return s;
  if (qDesc->nb != 4 || !same_shape(*qDesc, *oDesc) || qDesc->dims[0] != d.c.B || qDesc->dims[1] < 1 ||
      qDesc->dims[1] % d.c.heads != 0 || qDesc->dims[3] != d.c.D)
    return GRXDNN_STATUS_INVALID_VALUE;
  if (weights) {
    if (!weights_shape(*weightsDesc, d.c.B, d.c.heads, (int64_t)d.c.W * d.c.page))
      return GRXDNN_STATUS_INVALID_VALUE;
    if (!std::isfinite(weightDecay) || weightDecay < 0.0f) return GRXDNN_STATUS_INVALID_VALUE;
  }
  if (qDesc->type != kCacheDesc->type || oDesc->type != kCacheDesc->type) return GRXDNN_STATUS_NOT_SUPPORTED;
  d.H = qDesc->dims[1];
  // one query per sequence; (sequence, query head) pairs are counted in 32 bits
  if (qDesc->dims[2] != 1 || d.H / d.c.heads > 1024 || (int64_t)d.c.B * d.H > INT_MAX / 4)
    return GRXDNN_STATUS_NOT_SUPPORTED;
  if (d.c.B == 0) return GRXDNN_STATUS_SUCCESS;
  if (!half_rows(*qDesc) || !half_rows(*oDesc)) return GRXDNN_STATUS_NOT_SUPPORTED;
  if (!no_overlap(*oDesc) || (weights && !no_overlap(*weightsDesc))) return GRXDNN_STATUS_INVALID_VALUE;
  if (!q || !kCache || !vCache || !table || !lengths || !o) return GRXDNN_STATUS_INVALID_VALUE;
  if (!grxk::paged_attention_fits(d.c, d.H, weights != nullptr)) return GRXDNN_STATUS_NOT_SUPPORTED;
  const size_t need = grxk::paged_attention_workspace(d.c, d.H, weights != nullptr);
  if (workspaceBytes < need || (need && !workspace)) return GRXDNN_STATUS_INVALID_VALUE;
  if (may_alias(*oDesc, o, *qDesc, q) && !(o == q && same_strides(*oDesc, *qDesc)))
    return GRXDNN_STATUS_INVALID_VALUE;
  // What is written, against everything else that the call reads or writes.
  const Span so = span_of(*oDesc, o, 2), sw = weights ? span_of(*weightsDesc, weights, 4) : Span{0, 0};
  const Span ss = need ? bytes_at(workspace, (int64_t)need) : Span{0, 0};
  const Span in[] = {span_of(*kCacheDesc, kCache, 2), span_of(*vCacheDesc, vCache, 2),
                     span_of(*tableDesc, table, 4), bytes_at(lengths, 4ll * d.c.B)};
  for (const Span& x : in)
    if (intersect(so, x) || (weights && intersect(sw, x)) || (need && intersect(ss, x)))
      return GRXDNN_STATUS_INVALID_VALUE;
  const Span sq = span_of(*qDesc, q, 2);
  if (weights && (intersect(sw, so) || intersect(sw, sq))) return GRXDNN_STATUS_INVALID_VALUE;
  if (need && (intersect(ss, so) || intersect(ss, sq) || (weights && intersect(ss, sw))))
    return GRXDNN_STATUS_INVALID_VALUE;
  if (!aligned16(q) || !aligned16(kCache) || !aligned16(vCache) || !aligned16(o) ||
      (need && !aligned16(workspace)))
    return GRXDNN_STATUS_NOT_SUPPORTED;
  s = ensure_device(*handle);
  if (s != GRXDNN_STATUS_SUCCESS) return s;
  d.c.k = const_cast<void*>(kCache); d.c.v = const_cast<void*>(vCache);
  d.c.table = table; d.c.lengths = lengths;
  d.scale = attnDesc->scale;
  d.q = q; d.q_sb = qDesc->strides[0]; d.q_sh = qDesc->strides[1];
  d.o = o; d.o_sb = oDesc->strides[0]; d.o_sh = oDesc->strides[1];
  d.decay = weightDecay;
  if (weights) {
    d.weights = weights;
    d.w_sb = weightsDesc->strides[0];
    d.w_sh = weightsDesc->strides[1];
  }
  d.ws = workspace;
  return from_hip(grxk::launch_paged_attention(
      qDesc->type == GRX_R_16BF ? grxk::AttnType::BF16 : grxk::AttnType::F16, d, handle->stream));
}

grxdnnStatus_t grxdnnPagedCacheEvict(grxdnnHandle_t handle, grxdnnTensorDescriptor_t kCacheDesc, void* kCache,
                                     grxdnnTensorDescriptor_t vCacheDesc, void* vCache,
                                     grxdnnTensorDescriptor_t tableDesc, const int* table, const int* lengths,
                                     grxdnnTensorDescriptor_t weightsDesc, const float* weights, int budget,
                                     int recent, int* kept, grxdnnTensorDescriptor_t newTableDesc,
                                     const int* newTable, int* newLengths,
                                     grxdnnTensorDescriptor_t newWeightsDesc, float* newWeights) {
  if (!handle) return GRXDNN_STATUS_NOT_INITIALIZED;
  if (!weightsDesc || !newTableDesc || !newWeightsDesc || !weightsDesc->set || !newTableDesc->set ||
      !newWeightsDesc->set)
    return GRXDNN_STATUS_INVALID_VALUE;
  grxk::PagedEvictDesc d{};
  grxdnnStatus_t s = paged_cache(kCacheDesc, vCacheDesc, tableDesc, true, &d.c);
  if (s != GRXDNN_STATUS_SUCCESS) return s;
  if (budget < 1 || recent < 0 || recent > budget) return GRXDNN_STATUS_INVALID_VALUE;
  if (!table_shape(*newTableDesc) || newTableDesc->dims[0] != d.c.B ||
      (int64_t)newTableDesc->dims[1] * d.c.page < budget)
    return GRXDNN_STATUS_INVALID_VALUE;
  if ((int64_t)newTableDesc->dims[1] * d.c.page > kMaxRoom) return GRXDNN_STATUS_NOT_SUPPORTED;
  if (!weights_shape(*weightsDesc, d.c.B, d.c.heads, (int64_t)d.c.W * d.c.page) ||
      !weights_shape(*newWeightsDesc, d.c.B, d.c.heads, budget))
    return GRXDNN_STATUS_INVALID_VALUE;
  if (d.c.B == 0) return GRXDNN_STATUS_SUCCESS;
  if (!no_overlap(*newWeightsDesc)) return GRXDNN_STATUS_INVALID_VALUE;
  if (!kCache || !vCache || !table || !lengths || !weights || !kept || !newTable || !newLengths || !newWeights)
    return GRXDNN_STATUS_INVALID_VALUE;
  if (may_alias(*kCacheDesc, kCache, *vCacheDesc, vCache)) return GRXDNN_STATUS_INVALID_VALUE;
  // Each written array against everything else; the pools are read and written.
  const Span spans[] = {span_of(*kCacheDesc, kCache, 2), span_of(*vCacheDesc, vCache, 2),
                        bytes_at(kept, 4ll * d.c.B * d.c.heads * budget), bytes_at(newLengths, 4ll * d.c.B),
                        span_of(*newWeightsDesc, newWeights, 4),
                        // only read from here on
                        span_of(*tableDesc, table, 4), span_of(*newTableDesc, newTable, 4),
                        span_of(*weightsDesc, weights, 4), bytes_at(lengths, 4ll * d.c.B)};
  for (int i = 0; i < 5; ++i)
    for (int j = i + 1; j < 9; ++j) {
      if (i == 0 && j == 1) continue;                      // the pools: element by element, above
      if (i == 3 && j == 8 && newLengths == lengths) continue;   // in place
      if (intersect(spans[i], spans[j])) return GRXDNN_STATUS_INVALID_VALUE;
    }
  if (!aligned16(kCache) || !aligned16(vCache)) return GRXDNN_STATUS_NOT_SUPPORTED;
  s = ensure_device(*handle);
  if (s != GRXDNN_STATUS_SUCCESS) return s;
  d.c.k = kCache; d.c.v = vCache; d.c.table = table; d.c.lengths = lengths;
  d.weights = weights; d.w_sb = weightsDesc->strides[0]; d.w_sh = weightsDesc->strides[1];
  d.budget = budget; d.recent = recent; d.kept = kept;
  d.new_table = newTable; d.new_table_rs = newTableDesc->strides[0]; d.new_W = newTableDesc->dims[1];
  d.new_lengths = newLengths;
  d.new_weights = newWeights; d.nw_sb = newWeightsDesc->strides[0]; d.nw_sh = newWeightsDesc->strides[1];
  d.nw_slots = newWeightsDesc->dims[2];
  return from_hip(grxk::launch_paged_evict(d, handle->stream));
}

grxdnnStatus_t grxdnnTokenLogProbGetWorkspaceSize(grxdnnHandle_t handle, grxdnnTensorDescriptor_t xDesc,
                                                  int topCount, size_t* bytes) {
  if (!handle) return GRXDNN_STATUS_NOT_INITIALIZED;
  if (!xDesc || !xDesc->set || !bytes || topCount < 0) return GRXDNN_STATUS_INVALID_VALUE;
  grxk::NormType nt{};
  int64_t rows = 0, pitch = 0;
  const grxdnnStatus_t s = logit_rows(*xDesc, &nt, &rows, &pitch);
  if (s != GRXDNN_STATUS_SUCCESS) return s;
  const int vocab = xDesc->dims[xDesc->nb - 1];
  if (rows && topCount > vocab) return GRXDNN_STATUS_INVALID_VALUE;
  if (topCount > 64) return GRXDNN_STATUS_NOT_SUPPORTED;
  *bytes = rows ? grxk::token_logprob_workspace(nt, rows, vocab, topCount) : 0;
  return GRXDNN_STATUS_SUCCESS;
}

grxdnnStatus_t grxdnnTokenLogProbForward(grxdnnHandle_t handle, grxdnnTensorDescriptor_t xDesc, const void* x,
                                         const int* tokens, float* logProb, float* logSumExp, float* entropy,
                                         int topCount, float* topLogProb, int* topIndex, void* workspace,
                                         size_t workspaceBytes) {
  size_t need = 0;
  grxdnnStatus_t s = grxdnnTokenLogProbGetWorkspaceSize(handle, xDesc, topCount, &need);
  if (s != GRXDNN_STATUS_SUCCESS) return s;
  if ((tokens != nullptr) != (logProb != nullptr)) return GRXDNN_STATUS_INVALID_VALUE;
  if (topCount ? !topLogProb || !topIndex : topLogProb || topIndex) return GRXDNN_STATUS_INVALID_VALUE;
  grxk::NormType nt{};
  grxk::TokenLogProbDesc d{};
  (void)logit_rows(*xDesc, &nt, &d.rows, &d.x_row_stride);
  if (d.rows == 0) return GRXDNN_STATUS_SUCCESS;
  if (!x || !logSumExp) return GRXDNN_STATUS_INVALID_VALUE;
  if (workspaceBytes < need || (need && !workspace)) return GRXDNN_STATUS_INVALID_VALUE;
  // Each written array against the inputs and the other written ones.
  const Span spans[] = {logProb ? bytes_at(logProb, 4 * d.rows) : Span{0, 0},
                        bytes_at(logSumExp, 4 * d.rows),
                        entropy ? bytes_at(entropy, 4 * d.rows) : Span{0, 0},
                        topCount ? bytes_at(topLogProb, 4 * d.rows * topCount) : Span{0, 0},
                        topCount ? bytes_at(topIndex, 4 * d.rows * topCount) : Span{0, 0},
                        need ? bytes_at(workspace, (int64_t)need) : Span{0, 0},
                        span_of(*xDesc, x, element_size(nt)),
                        tokens ? bytes_at(tokens, 4 * d.rows) : Span{0, 0}};
  for (int i = 0; i < 6; ++i)
    for (int j = i + 1; j < 8; ++j)
      if (intersect(spans[i], spans[j])) return GRXDNN_STATUS_INVALID_VALUE;
  if (need && !aligned16(workspace)) return GRXDNN_STATUS_NOT_SUPPORTED;
  s = ensure_device(*handle);
  if (s != GRXDNN_STATUS_SUCCESS) return s;
  d.vocab = xDesc->dims[xDesc->nb - 1];
  d.x = x; d.tokens = tokens; d.logprob = logProb; d.lse = logSumExp; d.entropy = entropy;
  d.top = topCount; d.top_logprob = topLogProb; d.top_index = topIndex;
  d.ws = workspace;
  return from_hip(grxk::launch_token_logprob(nt, d, handle->stream));
}

grxdnnStatus_t grxdnnTokenLogProbBackward(grxdnnHandle_t handle, grxdnnTensorDescriptor_t xDesc, const void* x,
                                          const int* tokens, const float* logSumExp, const float* entropy,
                                          const float* dLogProb, const float* dEntropy,
                                          grxdnnTensorDescriptor_t dxDesc, void* dx) {
  if (!handle) return GRXDNN_STATUS_NOT_INITIALIZED;
  if (!xDesc || !dxDesc || !xDesc->set || !dxDesc->set) return GRXDNN_STATUS_INVALID_VALUE;
  if (!same_shape(*xDesc, *dxDesc)) return GRXDNN_STATUS_INVALID_VALUE;
  if ((tokens != nullptr) != (dLogProb != nullptr) || (dEntropy && !entropy) || (!tokens && !dEntropy))
    return GRXDNN_STATUS_INVALID_VALUE;
  if (xDesc->type != dxDesc->type) return GRXDNN_STATUS_NOT_SUPPORTED;
  grxk::NormType nt{};
  grxk::TokenLogProbGradDesc d{};
  int64_t rows = 0;
  grxdnnStatus_t s = logit_rows(*xDesc, &nt, &d.rows, &d.x_row_stride);
  if (s != GRXDNN_STATUS_SUCCESS) return s;
  s = logit_rows(*dxDesc, &nt, &rows, &d.dx_row_stride);
  if (s != GRXDNN_STATUS_SUCCESS) return s;
  if (d.rows == 0) return GRXDNN_STATUS_SUCCESS;
  if (!x || !logSumExp || !dx) return GRXDNN_STATUS_INVALID_VALUE;
  if (!no_overlap(*dxDesc)) return GRXDNN_STATUS_INVALID_VALUE;
  const Span out = span_of(*dxDesc, dx, element_size(nt));
  if (intersect(out, span_of(*xDesc, x, element_size(nt))) && !(dx == x && same_strides(*dxDesc, *xDesc)))
    return GRXDNN_STATUS_INVALID_VALUE;
  for (const void* p : {(const void*)tokens, (const void*)logSumExp, (const void*)entropy,
                        (const void*)dLogProb, (const void*)dEntropy})
    if (p && intersect(out, bytes_at(p, 4 * d.rows))) return GRXDNN_STATUS_INVALID_VALUE;
  s = ensure_device(*handle);
  if (s != GRXDNN_STATUS_SUCCESS) return s;
  d.vocab = xDesc->dims[xDesc->nb - 1];
  d.x = x; d.tokens = tokens; d.lse = logSumExp; d.entropy = dEntropy ? entropy : nullptr;
  d.dlogprob = dLogProb; d.dentropy = dEntropy; d.dx = dx;
  return from_hip(grxk::launch_token_logprob_grad(nt, d, handle->stream));
}

}  // extern "C"
#pragma GCC visibility pop
