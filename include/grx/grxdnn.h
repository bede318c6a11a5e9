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

/* ---- norm and rotation of queries and keys ----------------------------------
 *
 * What comes between a projection and attention, in one pass: every head's row of
 * D values normalised by itself, and turned by its token's position.
 *   n = x / sqrt(mean(x^2) + eps),  u = n * gamma     (without gains: u = x)
 *   y[j] = u[j] cos - u[j'] sin,  y[j'] = u[j'] cos + u[j] sin
 *                                 of positions[b,s] * inverseFrequencies[i]
 * for the i-th of rotaryDim / 2 pairs (j, j'): (i, i + rotaryDim / 2) for
 * GRXDNN_ROPE_HALVES, (2i, 2i + 1) for GRXDNN_ROPE_PAIRS. Values from rotaryDim on
 * are not turned.
 *
 * q, yq: [B, H, S, D] and k, yk: [B, Hkv, S, D] of one type (GRX_R_16BF, GRX_R_16F
 * or GRX_R_32F), any strides that are multiples of 16 bytes (views of a packed
 * projection, of [B, S, H, D] memory), innermost stride 1, pointers 16-byte
 * aligned; D is 64, 128 or 256, B * S at most 2^31 - 4096 and H + Hkv at most 2^20
 * (else NOT_SUPPORTED). qGamma, kGamma: [D] of that type, contiguous, described
 * by wDesc; wDesc and both NULL: no norm, and eps is not looked at. All key
 * arguments NULL together: queries alone. rotaryDim: 0 .. D in steps of 16;
 * 0: no rotation, positions and inverseFrequencies are not read and may be NULL
 * (norm or rotation: INVALID_VALUE for neither). positions: B * S ints, packed
 * (a decoding step's are the sequences' lengths before the token), negative ones
 * turn back; inverseFrequencies: rotaryDim / 2 fp32. Both are device memory, read
 * when the kernels run.
 *
 * Sums and products are fp32 and y is rounded once; angles are reduced from the
 * whole product (64 bits and its remainder), for |angle| < 2^40. A row whose sum
 * of squares exceeds fp32's range is scaled by 0; mean(x^2) + eps is to be 2^-126 or
 * more (a row of zeros with eps 0 is NaN, as in the formula). Outputs must not share elements
 * of their own or with each other or with what the call reads, but yq may be q
 * and yk k (same pointer and strides); else INVALID_VALUE.
 * (New: planned by ref docs/designs/grxcp_roadmap.md:864-877.) */
typedef enum {
  GRXDNN_ROPE_HALVES = 0,
  GRXDNN_ROPE_PAIRS  = 1
} grxdnnRopeMode_t;

grxdnnStatus_t grxdnnQkNormRopeForward(grxdnnHandle_t handle,
                                       grxdnnTensorDescriptor_t qDesc, const void* q,
                                       grxdnnTensorDescriptor_t kDesc, const void* k,
                                       grxdnnTensorDescriptor_t wDesc, const void* qGamma,
                                       const void* kGamma, float eps,
                                       grxdnnRopeMode_t mode, int rotaryDim,
                                       const int* positions, const float* inverseFrequencies,
                                       grxdnnTensorDescriptor_t yqDesc, void* yq,
                                       grxdnnTensorDescriptor_t ykDesc, void* yk);

/* The gradient of that, from the forward call's inputs and the gradients dyq, dyk of
 * its outputs. With g the row of dy turned back:
 *   dx = r (g gamma - n mean(g gamma n)),  r = 1 / sqrt(mean(x^2) + eps)     (without gains: dx = g)
 *   dqGamma[j] = sum over b, h, s of g[j] n[j],  and dkGamma over the keys' rows
 * dyq, dq: [B, H, S, D], dyk, dk: [B, Hkv, S, D], of the inputs' type and rules; dq may
 * be dyq and dk dyk (same pointer and strides), or q and k. dqGamma, dkGamma: D fp32
 * each, overwritten, packed; NULL for what is not asked for, and without gains. Without
 * gains q and k are not read and may be NULL (their descriptors are needed). Sums are
 * fp32, in an order that does not change from call to call.
 * workspace: device memory of at least the size that
 * grxdnnQkNormRopeGetWorkspaceSize gives for the same descriptors (kDesc NULL
 * without keys; 0 bytes without wDesc), 16-byte aligned; needed where dqGamma or
 * dkGamma is asked for. Calls that may run at the same time, captured graphs
 * included, need workspaces of their own. */
grxdnnStatus_t grxdnnQkNormRopeGetWorkspaceSize(grxdnnHandle_t handle,
                                                grxdnnTensorDescriptor_t qDesc,
                                                grxdnnTensorDescriptor_t kDesc,
                                                grxdnnTensorDescriptor_t wDesc, size_t* bytes);
grxdnnStatus_t grxdnnQkNormRopeBackward(grxdnnHandle_t handle,
                                        grxdnnTensorDescriptor_t qDesc, const void* q,
                                        grxdnnTensorDescriptor_t kDesc, const void* k,
                                        grxdnnTensorDescriptor_t wDesc, const void* qGamma,
                                        const void* kGamma, float eps,
                                        grxdnnRopeMode_t mode, int rotaryDim,
                                        const int* positions, const float* inverseFrequencies,
                                        grxdnnTensorDescriptor_t dyqDesc, const void* dyq,
                                        grxdnnTensorDescriptor_t dykDesc, const void* dyk,
                                        grxdnnTensorDescriptor_t dqDesc, void* dq,
                                        grxdnnTensorDescriptor_t dkDesc, void* dk,
                                        float* dqGamma, float* dkGamma,
                                        void* workspace, size_t workspaceBytes);

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

/* ---- paged key-value cache in 8 bits ----------------------------------------
 *
 * The cache above with pools of GRX_R_8I codes: half the memory and half of what
 * attention reads. A code c of a block of slots stands for c * scale of the block:
 * scales are GRX_R_32F [pages, Hkv, N], any strides, N a divisor of P, so that row r of
 * a page belongs to block r / (P / N) (N = P: a scale for each slot; 1: one for the
 * page's). kScale and vScale are of one descriptor. Blocks have 1 .. 256 slots (else
 * NOT_SUPPORTED). The pools' strides but the last are multiples of 16 elements; what
 * is said above of tables, lengths, entries and overlaps holds, and D is 64 or 128.
 * (New: planned by ref docs/designs/grxcp_roadmap.md:864-877, "attention".) */

/* New rows behind the tokens that the cache holds, as grxdnnPagedCacheAppend puts
 * them, in 8 bits. For every block of every head that gets rows, keys and values each:
 *   need   = the least number of 8 significant bits (and at least 2^-126) that is not
 *            below max |x| / 127 over the block's new rows; 0 where all are 0, NaN where
 *            one is infinite or NaN
 *   scale' = max(scale, need) where the block holds rows of the sequence already
 *            (NaN if one of the two is), else need: what scale held before is not looked at
 *   code   = x / scale' to the nearest whole number, ties to the even one
 * and, where scale' > scale, the codes of rows that it holds already become code *
 * scale / scale', rounded so. Where scale' is 0 or not finite the new rows' codes are 0 and
 * the others stay: with NaN the whole block reads as NaN until it is begun anew. Rows
 * behind the new ones are left as they are.
 * Slots of a block that another sequence shares must not be followed by rows of this
 * call (they would be rounded again): share whole blocks.
 * A block that two written table entries name may hold codes of one and the scale of
 * another: what it reads as is none of the values written.
 * k, v: [B, Hkv, T, D], GRX_R_16BF or GRX_R_16F, counts as in grxdnnPagedCacheAppend;
 * (T + 512) * Hkv below 2^31. Scales that the caller sets are finite and >= 0. */
grxdnnStatus_t grxdnnPagedCacheAppendQuantized(grxdnnHandle_t handle,
                                               grxdnnTensorDescriptor_t kDesc, const void* k,
                                               grxdnnTensorDescriptor_t vDesc, const void* v,
                                               grxdnnTensorDescriptor_t kCacheDesc, void* kCache,
                                               grxdnnTensorDescriptor_t vCacheDesc, void* vCache,
                                               grxdnnTensorDescriptor_t scaleDesc, float* kScale,
                                               float* vScale,
                                               grxdnnTensorDescriptor_t tableDesc, const int* table,
                                               const int* lengths, const int* counts);

/* Rows of such a cache: for every sequence b, head h and t < T,
 *   k[b, h, t, :] = scale * code of slot first[b] + t      (and v)
 * and 0 where that slot is at or past lengths[b] or on a page that does not exist.
 * first: B ints (below 0 counts as 0), or NULL for 0 each. k, v: [B, Hkv, T, D] of
 * GRX_R_16BF, GRX_R_16F or GRX_R_32F, strides multiples of 16 bytes, T * Hkv at most
 * 2^31 - 4096; rounded once; what is past the type's range comes back as its largest
 * value. To go on in a cache of 16 bits (grxdnnPagedCacheAppend), which eviction needs, or
 * for grxdnnAttentionForward over a whole prompt (as many heads and tokens as queries). */
grxdnnStatus_t grxdnnPagedCacheReadQuantized(grxdnnHandle_t handle,
                                             grxdnnTensorDescriptor_t kCacheDesc, const void* kCache,
                                             grxdnnTensorDescriptor_t vCacheDesc, const void* vCache,
                                             grxdnnTensorDescriptor_t scaleDesc, const float* kScale,
                                             const float* vScale,
                                             grxdnnTensorDescriptor_t tableDesc, const int* table,
                                             const int* lengths, const int* first,
                                             grxdnnTensorDescriptor_t kDesc, void* k,
                                             grxdnnTensorDescriptor_t vDesc, void* v);

/* Attention of one new token per sequence over such a cache: grxdnnPagedAttentionForward
 * without weights, with the slots' codes times their scales for keys and values.
 * q, o: [B, H, 1, D], GRX_R_16BF or GRX_R_16F; its rules and limits hold. A query's row is
 * taken to 2^-22 of its largest value (or to 2^-127), products with the codes are
 * exact, scores, softmax and sums fp32 (a weight below 2^-126 of the largest counts as 0). A
 * weight times its slot's scale of a value keeps 21 bits, or 2^-36 of the query's largest such
 * product where that is more, and o is rounded once. A row of q with NaN or infinities in
 * it gives NaN, and so does a head of a sequence with a scale of NaN among its slots'
 * blocks. Values' scales up to 2^95.
 * workspace: as there, of grxdnnPagedAttentionQuantizedGetWorkspaceSize. */
grxdnnStatus_t grxdnnPagedAttentionQuantizedGetWorkspaceSize(grxdnnHandle_t handle,
                                                             grxdnnTensorDescriptor_t qDesc,
                                                             grxdnnTensorDescriptor_t kCacheDesc,
                                                             grxdnnTensorDescriptor_t tableDesc,
                                                             size_t* bytes);
grxdnnStatus_t grxdnnPagedAttentionQuantizedForward(grxdnnHandle_t handle,
                                                    grxdnnAttentionDescriptor_t attnDesc,
                                                    grxdnnTensorDescriptor_t qDesc, const void* q,
                                                    grxdnnTensorDescriptor_t kCacheDesc, const void* kCache,
                                                    grxdnnTensorDescriptor_t vCacheDesc, const void* vCache,
                                                    grxdnnTensorDescriptor_t scaleDesc, const float* kScale,
                                                    const float* vScale,
                                                    grxdnnTensorDescriptor_t tableDesc, const int* table,
                                                    const int* lengths,
                                                    grxdnnTensorDescriptor_t oDesc, void* o,
                                                    void* workspace, size_t workspaceBytes);

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
