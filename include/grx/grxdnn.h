/* grxdnn.h -- grxDNN primitives, MI355X (gfx950) build.
 *
 * The reference plans grxDNN but ships no code for it: a CMake slot
 * (ref: src/libs/CMakeLists.txt:12), an architecture entry naming grxdnn.h
 * (ref: docs/designs/grxcp_architecture.md:594, 640) and roadmap phase 6
 * (ref: docs/designs/grxcp_roadmap.md:864-877: "softmax, layernorm, ...,
 * attention; grxBLAS + custom kernels"). This header is therefore designed
 * new, in grxBLAS's style (ref: include/grx/grxblas.h): an opaque handle with
 * a borrowed stream, status codes with grxBLAS's values, device pointers for
 * tensors, host values for scalars, asynchronous calls, validation before any
 * device work and NOT_SUPPORTED instead of a silent fallback.
 *
 * Tensors are described cuDNN-style by an N-d descriptor (type, dims,
 * strides in elements). The innermost dimension must have stride 1.
 */
#ifndef GRXDNN_H
#define GRXDNN_H

#include "grx_cycles.h"
#include "grx_runtime.h"
#include "grx_types.h"

#ifdef __cplusplus
extern "C" {
#endif

typedef struct grxdnnContext*          grxdnnHandle_t;
typedef struct grxdnnTensorStruct*     grxdnnTensorDescriptor_t;
typedef struct grxdnnAttentionStruct*  grxdnnAttentionDescriptor_t;

/* Same values as grxblasStatus_t (ref include/grx/grxblas.h:37-46). */
typedef enum {
  GRXDNN_STATUS_SUCCESS          = 0,
  GRXDNN_STATUS_NOT_INITIALIZED  = 1,
  GRXDNN_STATUS_ALLOC_FAILED     = 2,
  GRXDNN_STATUS_INVALID_VALUE    = 3,
  GRXDNN_STATUS_ARCH_MISMATCH    = 4,
  GRXDNN_STATUS_EXECUTION_FAILED = 5,
  GRXDNN_STATUS_NOT_SUPPORTED    = 6,
  GRXDNN_STATUS_INTERNAL_ERROR   = 7
} grxdnnStatus_t;

#define GRXDNN_DIM_MAX 8

const char* grxdnnGetStatusString(grxdnnStatus_t s);

grxdnnStatus_t grxdnnCreate   (grxdnnHandle_t* handle);
grxdnnStatus_t grxdnnDestroy  (grxdnnHandle_t handle);
grxdnnStatus_t grxdnnSetStream(grxdnnHandle_t handle, grxStream_t stream);
grxdnnStatus_t grxdnnGetStream(grxdnnHandle_t handle, grxStream_t* stream);

/* ---- tensor descriptors ------------------------------------------------- */
grxdnnStatus_t grxdnnCreateTensorDescriptor (grxdnnTensorDescriptor_t* desc);
grxdnnStatus_t grxdnnDestroyTensorDescriptor(grxdnnTensorDescriptor_t desc);
/* 1 <= nbDims <= GRXDNN_DIM_MAX; dims >= 0; strides >= 0 in elements.
 * strides may be NULL for a packed (row-major, last dimension contiguous)
 * layout. */
grxdnnStatus_t grxdnnSetTensorNdDescriptor(grxdnnTensorDescriptor_t desc,
                                           grxDataType_t dataType, int nbDims,
                                           const int dims[],
                                           const int strides[]);
grxdnnStatus_t grxdnnGetTensorNdDescriptor(grxdnnTensorDescriptor_t desc,
                                           int nbDimsRequested,
                                           grxDataType_t* dataType,
                                           int* nbDims, int dims[],
                                           int strides[]);

/* ---- normalisation ------------------------------------------------------
 * x, y: [..., hidden]; every dimension but the last is a row index, the last
 * is normalised. The row dimensions must flatten to one row stride (packed
 * rows, or rows padded by a constant pitch). gamma/beta: 1-d [hidden],
 * contiguous, same type as x. Supported types: GRX_R_16BF, GRX_R_16F,
 * GRX_R_32F, with y of the same type and shape as x. Reductions are fp32.
 *
 *   RMSNorm:   y = x * rsqrt(mean(x^2) + eps) * gamma
 *   LayerNorm: y = (x - mean(x)) * rsqrt(var(x) + eps) * gamma + beta
 *              (biased variance)
 * eps must be finite and >= 0. hidden must be >= 1 and <= 65536. */
grxdnnStatus_t grxdnnRMSNormForward(grxdnnHandle_t handle,
                                    grxdnnTensorDescriptor_t xDesc,
                                    const void* x,
                                    grxdnnTensorDescriptor_t wDesc,
                                    const void* gamma, float eps,
                                    grxdnnTensorDescriptor_t yDesc, void* y);

grxdnnStatus_t grxdnnLayerNormForward(grxdnnHandle_t handle,
                                      grxdnnTensorDescriptor_t xDesc,
                                      const void* x,
                                      grxdnnTensorDescriptor_t wDesc,
                                      const void* gamma, const void* beta,
                                      float eps,
                                      grxdnnTensorDescriptor_t yDesc, void* y);

/* ---- softmax (forward) ---------------------------------------------------
 * Over the last dimension of x, every other dimension a row index:
 *   y[..., i] = exp(x[..., i] - m) / sum_j exp(x[..., j] - m),  m = max_j x[..., j]
 * Same layout rules and types as the normalisations above (rows flatten to
 * one row stride, innermost stride 1; GRX_R_16BF, GRX_R_16F or GRX_R_32F; y
 * of x's type and shape); fp32 arithmetic, y rounded once. A row whose every
 * element is -inf gives NaN, as the formula does. hidden: 1 .. 2^24.
 * (New: planned by ref docs/designs/grxcp_roadmap.md:864-877.) */
grxdnnStatus_t grxdnnSoftmaxForward(grxdnnHandle_t handle,
                                    grxdnnTensorDescriptor_t xDesc, const void* x,
                                    grxdnnTensorDescriptor_t yDesc, void* y);

/* ---- GELU (forward, element-wise) -----------------------------------------
 *   GRXDNN_GELU_ERF:  y = x/2 * (1 + erf(x / sqrt(2)))
 *   GRXDNN_GELU_TANH: y = x/2 * (1 + tanh(sqrt(2/pi) * (x + 0.044715 x^3)))
 * x and y: descriptors of the same shape and type (GRX_R_16BF, GRX_R_16F,
 * GRX_R_32F) under the row layout rules above; fp32 arithmetic, y rounded
 * once; y may be x (in place). hidden: 1 .. 2^24.
 * (New: planned by ref docs/designs/grxcp_roadmap.md:864-877.) */
typedef enum {
  GRXDNN_GELU_ERF  = 0,
  GRXDNN_GELU_TANH = 1
} grxdnnGeluMode_t;

grxdnnStatus_t grxdnnGeluForward(grxdnnHandle_t handle, grxdnnGeluMode_t mode,
                                 grxdnnTensorDescriptor_t xDesc, const void* x,
                                 grxdnnTensorDescriptor_t yDesc, void* y);

/* ---- fused scaled-dot-product attention (forward) ----------------------
 *
 *   O[b,h,i,:] = sum_j softmax_j( scale * <Q[b,h,i,:], K[b,h,j,:]> + mask ) V[b,h,j,:]
 *
 * with mask = -inf for j > i when causal (the query and key sequences have
 * the same length and are aligned at position 0). Q, K, V, O are 4-d
 * [B, H, S, D] descriptors of one type (GRX_R_16BF or GRX_R_16F), innermost
 * stride 1, with equal B, H, S and D. Supported head dimensions: 64, 128.
 * The other strides are multiples of 8 elements and the pointers 16-byte
 * aligned, and each tensor's sequence stride times 2 * (S + 256) bytes stays
 * below 2^31 (else NOT_SUPPORTED); O's elements must not share addresses (else
 * INVALID_VALUE), while Q, K and V may (a broadcast). O must share no
 * element with K or V, and none with Q unless it is Q itself (same pointer,
 * same strides: in place); else INVALID_VALUE. Where O and the other view
 * have the same strides the test is exact, element by element (O in its own
 * slot of a packed [B, S, n, H, D] buffer is accepted); otherwise it is on
 * the address ranges the descriptors span.
 * Softmax and both products accumulate in fp32; O is rounded once (RNE). */
grxdnnStatus_t grxdnnCreateAttentionDescriptor (grxdnnAttentionDescriptor_t* d);
grxdnnStatus_t grxdnnDestroyAttentionDescriptor(grxdnnAttentionDescriptor_t d);
/* causal: 0 or 1. softmaxScale: finite and > 0 (1/sqrt(D) is the usual). */
grxdnnStatus_t grxdnnSetAttentionDescriptor(grxdnnAttentionDescriptor_t d,
                                            int causal, float softmaxScale);
grxdnnStatus_t grxdnnGetAttentionDescriptor(grxdnnAttentionDescriptor_t d,
                                            int* causal, float* softmaxScale);

grxdnnStatus_t grxdnnAttentionForward(grxdnnHandle_t handle,
                                      grxdnnAttentionDescriptor_t attnDesc,
                                      grxdnnTensorDescriptor_t qDesc, const void* q,
                                      grxdnnTensorDescriptor_t kDesc, const void* k,
                                      grxdnnTensorDescriptor_t vDesc, const void* v,
                                      grxdnnTensorDescriptor_t oDesc, void* o);

/* Per-wave cycle records of grxdnnAttentionForward, in grxBLAS's probe
 * format and manner (grx_cycles.h; ref include/grx/grxblas.h:240-242, which
 * grxDNN, new, extends to attention). With a slot array attached, the next
 * attention calls write one grxCycleSlot per wave that has work (slot =
 * workgroup * waves per workgroup + wave; s_memtime at entry and exit, core
 * = XCD << 16 | CU id); capacity must cover
 * grxdnnAttentionCycleSlotsNeeded for the call's B, H and S, else the call
 * returns INVALID_VALUE before any device work. NULL turns recording off.
 * A recorded call always runs the persistent kernel that the slots are counted
 * for, also where the call alone would split its keys over workgroups of fewer
 * queries. */
grxdnnStatus_t grxdnnSetCycleProbe(grxdnnHandle_t handle, grxCycleSlot* slots,
                                   int capacity);
int            grxdnnAttentionCycleSlotsNeeded(grxdnnHandle_t handle, int batch,
                                               int heads, int seqLen);

/* ---- paged key-value cache --------------------------------------------------
 *
 * Keys and values of running sequences lie in two pools, each described by a
 * 4-d descriptor [pages, Hkv, P, D]: pages of P slots for Hkv heads of D values
 * (any strides: [pages, P, Hkv, D] memory is a view of it). A page table, 2-d
 * [B, W] GRX_R_32I with innermost stride 1, names the pages of each of B
 * sequences: slot j of sequence b is row j % P of page table[b][j / P], and a
 * sequence has room for W * P slots (at most 2^31 - 4096). lengths: B ints, the
 * slots of each sequence that hold tokens; below 0 counts as 0, above W * P as
 * W * P. Tables, lengths and counts are device memory, read when the kernels
 * run: a captured call follows their contents on every replay, and they must not
 * change while a call that reads them runs.
 *
 * Table entries of pages that a call does not reach are not read. An entry
 * outside [0, pages) that it does reach is never followed: a row written there
 * is dropped, and a row read there is as if the slot were not in the sequence.
 * Two sequences may share pages that are only read.
 *
 * Types GRX_R_16BF or GRX_R_16F, one for all key, value, query and output
 * tensors; D is 64 or 128; innermost stride 1, the other strides multiples of 8
 * elements, pointers 16-byte aligned, B * Hkv below 2^29 (else NOT_SUPPORTED).
 * The two pools have one shape and share no element; written tensors must not
 * share elements of their own or with what the call reads (INVALID_VALUE where
 * the descriptors show it; pages that two written table entries name are the
 * caller's matter: such rows hold one of the values written).
 * (New: planned by ref docs/designs/grxcp_roadmap.md:864-877, "attention".) */

/* New rows behind the tokens that a cache holds: for every sequence b, head h
 * and t < counts[b],
 *   cache[slot lengths[b] + t of b, head h] = new[b, h, t, :]   (keys and values)
 * k, v: [B, Hkv, T, D]. counts: B ints within 0 .. T (others are clamped), or
 * NULL for T each. Rows past a sequence's room are dropped. lengths is not
 * changed: the caller adds counts to it. */
grxdnnStatus_t grxdnnPagedCacheAppend(grxdnnHandle_t handle,
                                      grxdnnTensorDescriptor_t kDesc, const void* k,
                                      grxdnnTensorDescriptor_t vDesc, const void* v,
                                      grxdnnTensorDescriptor_t kCacheDesc, void* kCache,
                                      grxdnnTensorDescriptor_t vCacheDesc, void* vCache,
                                      grxdnnTensorDescriptor_t tableDesc, const int* table,
                                      const int* lengths, const int* counts);

/* Attention of one new token per sequence over its slots (the token's own key
 * and value included, appended before):
 *   s[b,h,j] = softmaxScale * <q[b,h,0,:], K[slot j of b, head h / G, :]>,  j < lengths[b]
 *   p[b,h,:] = softmax(s[b,h,:]),  o[b,h,0,:] = sum_j p[b,h,j] V[slot j of b, head h / G, :]
 * q, o: [B, H, 1, D], H = G * Hkv query heads in groups of G = 1 .. 1024. The
 * descriptor's causal flag makes no difference: the new token is the last one.
 * Scores, softmax and sums are fp32, the weights of the values keep 16 bits (bf16)
 * or 21 (f16), and o is rounded once. o may be q itself (same pointer and
 * strides). A sequence of no slots gives o = 0; one whose scores are all -inf
 * gives NaN, as the formula does. Slots at or past lengths[b] are not read,
 * whatever their pages hold.
 *
 * weights (optional, both arguments or neither NULL): what the slots received,
 * [B, Hkv, S] GRX_R_32F, S >= W * P, innermost stride 1:
 *   weights[b,g,j] = weightDecay * weights[b,g,j] + sum_{h in group g} p[b,h,j],  j < lengths[b]
 * with entries at or past lengths[b] left as they are. weightDecay: finite and
 * >= 0; with 0 the old weights are not read. Nothing else adds to them: what a
 * prompt's tokens gave each other (grxdnnAttentionForward) is not in them, so the
 * slots of a prompt are equal before the first call.
 *
 * B * Hkv * ceil(G / 32) * W * P below 2^36, B * H below 2^29, and with weights
 * Hkv * ceil(W * P / 1024) + H below 2^24 (else NOT_SUPPORTED, and nothing is
 * launched).
 *
 * workspace: device memory of at least the size that
 * grxdnnPagedAttentionGetWorkspaceSize gives for the same descriptors (a
 * smaller one is INVALID_VALUE; 16-byte aligned; its contents before the call
 * do not matter). Calls that may run at the same time, captured graphs
 * included, need workspaces of their own. */
grxdnnStatus_t grxdnnPagedAttentionGetWorkspaceSize(grxdnnHandle_t handle,
                                                    grxdnnTensorDescriptor_t qDesc,
                                                    grxdnnTensorDescriptor_t kCacheDesc,
                                                    grxdnnTensorDescriptor_t tableDesc,
                                                    grxdnnTensorDescriptor_t weightsDesc,
                                                    size_t* bytes);
grxdnnStatus_t grxdnnPagedAttentionForward(grxdnnHandle_t handle,
                                           grxdnnAttentionDescriptor_t attnDesc,
                                           grxdnnTensorDescriptor_t qDesc, const void* q,
                                           grxdnnTensorDescriptor_t kCacheDesc, const void* kCache,
                                           grxdnnTensorDescriptor_t vCacheDesc, const void* vCache,
                                           grxdnnTensorDescriptor_t tableDesc, const int* table,
                                           const int* lengths, float weightDecay,
                                           grxdnnTensorDescriptor_t weightsDesc, float* weights,
                                           grxdnnTensorDescriptor_t oDesc, void* o,
                                           void* workspace, size_t workspaceBytes);

/* The slots of each sequence and head that matter, into pages of their own. Of
 * n = lengths[b] slots with weights[b,h,:] (as grxdnnPagedAttentionForward
 * accumulates them) head h of sequence b keeps all if n <= budget, else the
 * newest `recent` ones (0 <= recent <= budget) and, of the others, the
 * budget - recent of largest weight; of equal weights the lower slots stay, -0
 * equals 0 and NaN counts as largest. With m = min(n, budget), in slot order:
 *   kept[b,h,i]       = slot of the i-th one,       -1 for i >= m
 *   row i of the sequence in newTable = that slot's key and value,  i < m
 *   newWeights[b,h,i] = its weight,                  0 for i >= m
 *   newLengths[b]     = m
 * table, newTable: [B, W] and [B, W2] (any W2 * P >= budget) over the same pools;
 * pages named by newTable must not be pages that any sequence of the call
 * reads (a page may be shared by sequences: their rows are copied out of it).
 * The pages of table are the caller's again afterwards. kept: packed
 * [B, Hkv, budget] ints. weights, newWeights: [B, Hkv, S], S >= W * P and
 * [B, Hkv, S2], S2 >= budget, GRX_R_32F, innermost stride 1. newLengths may be
 * lengths itself. budget >= 1. A slot on a page that does not exist is kept or not
 * by its weight like the others; its row of newTable is left as it was, and counts
 * as a slot from then on. */
grxdnnStatus_t grxdnnPagedCacheEvict(grxdnnHandle_t handle,
                                     grxdnnTensorDescriptor_t kCacheDesc, void* kCache,
                                     grxdnnTensorDescriptor_t vCacheDesc, void* vCache,
                                     grxdnnTensorDescriptor_t tableDesc, const int* table,
                                     const int* lengths,
                                     grxdnnTensorDescriptor_t weightsDesc, const float* weights,
                                     int budget, int recent, int* kept,
                                     grxdnnTensorDescriptor_t newTableDesc, const int* newTable,
                                     int* newLengths,
                                     grxdnnTensorDescriptor_t newWeightsDesc, float* newWeights);

/* ---- log probabilities of tokens ---------------------------------------------
 * x: logits [..., V] under softmax's layout rules and types (rows flatten to one
 * row stride; GRX_R_16BF, GRX_R_16F, GRX_R_32F; V = 1 .. 2^24). For row r of the R:
 *   logSumExp[r] = log sum_j exp(x[r,j])
 *   logProb[r]   = x[r, tokens[r]] - logSumExp[r]    (from the row's maximum, not the
 *                                                     rounded logSumExp; 0 where tokens[r] is
 *                                                     outside [0, V): a padded row)
 *   entropy[r]   = - sum_j p[r,j] log p[r,j],  p = softmax(x[r,:]),  0 log 0 = 0
 *   topLogProb[r,i], topIndex[r,i]: the i-th largest x[r,j] - logSumExp[r] and its j,
 *                  i < topCount; of equal ones the lower j comes first, -0 equals 0, NaN is largest
 * Device arrays, packed: tokens and topIndex 32-bit ints, the others fp32; sums
 * are fp32. entropy may be NULL, tokens and logProb may both be NULL; topCount
 * is 0 .. min(V, 64), the two top arrays NULL if 0. -inf (a masked token) has
 * p = 0. A row of only -inf has logSumExp -inf and NaN for the rest; one with NaN
 * or +inf in it is NaN throughout (inf - inf, as in softmax) but for topIndex and
 * the 0 of a padded row.
 * workspace: as for grxdnnPagedAttentionForward. */
grxdnnStatus_t grxdnnTokenLogProbGetWorkspaceSize(grxdnnHandle_t handle,
                                                  grxdnnTensorDescriptor_t xDesc, int topCount,
                                                  size_t* bytes);
grxdnnStatus_t grxdnnTokenLogProbForward(grxdnnHandle_t handle,
                                         grxdnnTensorDescriptor_t xDesc, const void* x,
                                         const int* tokens, float* logProb, float* logSumExp,
                                         float* entropy, int topCount, float* topLogProb,
                                         int* topIndex, void* workspace, size_t workspaceBytes);

/* The gradient of the log probabilities and entropies in the logits, from the
 * forward call's logSumExp and entropy:
 *   dx[r,j] = dLogProb[r] (1[j = tokens[r]] - p[r,j])         (0 without a token)
 *           - dEntropy[r] p[r,j] (log p[r,j] + entropy[r])    (0 where p = 0)
 * with p[r,j] = exp(x[r,j] - logSumExp[r]) (below 2^-126: 0). A row without a token
 * whose dEntropy is 0 or left out gets 0 whatever it holds: padding. tokens and
 * dLogProb may be NULL together, and dEntropy may be (entropy is then not read):
 * that term is left out; not both. dx: a descriptor of x's shape and type; fp32
 * arithmetic, rounded once; dx may be x itself (same pointer and strides).
 * topLogProb has no gradient here. */
grxdnnStatus_t grxdnnTokenLogProbBackward(grxdnnHandle_t handle,
                                          grxdnnTensorDescriptor_t xDesc, const void* x,
                                          const int* tokens, const float* logSumExp,
                                          const float* entropy, const float* dLogProb,
                                          const float* dEntropy,
                                          grxdnnTensorDescriptor_t dxDesc, void* dx);

#ifdef __cplusplus
}  /* extern "C" */
#endif

#endif  /* GRXDNN_H */
