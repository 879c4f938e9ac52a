/* SPDX-License-Identifier: Apache-2.0
 *
 * vccl-b200 model operators around a paged key/value cache held in 4 bits
 * (additions; no counterpart in the reference C API).
 *
 * All calls are stream-ordered on the device that is current, take device
 * pointers and allocate nothing: scratch is passed in (sizes from the
 * *Workspace calls), so a call may be captured into a CUDA graph.  Activation
 * tensors are vcclBfloat16 or vcclFloat16; [T, heads, D] tensors have
 * contiguous channels, and token and head strides (in elements, below 2^31)
 * that are multiples of 8 on a 16-byte aligned base; at most 32768 heads and
 * 2^30 tokens.
 *
 * The cache of one layer: uint8 [pages, kvHeads, pageSize / 16, 18 * D] with
 * pageSize a multiple of 16 and D 64 or 128.  A block of 16 tokens holds the
 * key codes (16 rows of D / 2 bytes), the value codes, then for each token
 * and 64 channels a bf16 scale and a bf16 midpoint of the keys, then of the
 * values:  value = midpoint + scale * (code - 7.5).  csrc/kernels/kv4.cuh
 * gives the order of channels inside a row.  A slot is page * pageSize +
 * place in the page; a negative slot, or one behind the cache, is skipped.
 */
#ifndef VCCL_MODEL_H_
#define VCCL_MODEL_H_

#include "vccl.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Block tables and slots from request lengths.  For request i of batch:
 * L_i = finished[i] ? 0 : lens[i] (finished may be NULL) and n_i =
 * max(newLens[i], 0) new tokens.  Finished requests give the
 * ceil(lens[i] / pageSize) pages of their table row back to the stack
 * freePages[0, *freeCount) (room for poolSize entries), in order; then
 * requests take ceil((L_i + n_i) / pageSize) - ceil(L_i / pageSize) pages
 * each from its top.  A request is granted if it fits the table (width
 * pages), its rows fit in the batch (tokens rows), and it needs no page or
 * the pages asked for up to and including it (those of refused requests
 * counted) are there.  Written: table and freePages in place;
 * qStarts[batch + 1] = prefix sums of n; kvLens[i] = granted ? L_i + n_i : 0;
 * lensOut[i] = L_i + (granted ? n_i : 0); *countOut; and for each of the
 * tokens rows its position, slot (-1 if refused or behind the last row) and
 * request (-1 behind the last row).  lensOut may be lens, countOut may be
 * freeCount.  scratch: 2 * batch + 1 words.  batch <= 8192. */
vcclResult_t vcclPagePlan(const int* lens, const int* newLens, const unsigned char* finished, int* table,
                          int* freePages, const int* freeCount, int batch, int width, int poolSize, int pageSize,
                          int tokens, int* positions, int* slots, int* requests, int* qStarts, int* kvLens,
                          int* lensOut, int* countOut, int* scratch, vcclStream_t stream);

/* A [tokens, heads, D] tensor: pointer and strides in elements. */
typedef struct {
  void* data;
  long long tokenStride;
  long long headStride;
  int heads;
} vcclHeads_t;

/* Norm and rotation of every head: x^ = x / sqrt(mean(x^2) + eps) * weight
 * where a weight [D] is given (else x^ = x), then the first 2 * half channels
 * rotate by positions[t] * invFreq[j] (f32 [half]; the angle is taken in 64
 * bits): channels (j, j + half), or (2j, 2j + 1) with interleaved != 0.
 * D % 8 == 0, D <= 256, half % 8 == 0, half >= 8, 2 * half <= D. */
typedef struct {
  const int* positions;
  const float* invFreq;
  const void* qWeight;
  const void* kWeight;
  int half;
  int interleaved;
  float eps;
} vcclRope_t;

/* qOut, kOut = norm and rotation of q, k; an output may be its input. */
vcclResult_t vcclQkNormRope(const vcclHeads_t* q, const vcclHeads_t* k, const vcclRope_t* rope,
                            const vcclHeads_t* qOut, const vcclHeads_t* kOut, int tokens, int D,
                            vcclDataType_t datatype, vcclStream_t stream);

/* Gradients of vcclQkNormRope: dqIn, dkIn from dq, dk (gradients of its
 * outputs) and q, k (its inputs); dqWeight, dkWeight [D] where rope has the
 * weights.  workspace: vcclQkNormRopeBackwardWorkspace bytes. */
size_t vcclQkNormRopeBackwardWorkspace(int D);
vcclResult_t vcclQkNormRopeBackward(const vcclHeads_t* dq, const vcclHeads_t* dk, const vcclHeads_t* q,
                                    const vcclHeads_t* k, const vcclRope_t* rope, const vcclHeads_t* dqIn,
                                    const vcclHeads_t* dkIn, void* dqWeight, void* dkWeight, void* workspace,
                                    int tokens, int D, vcclDataType_t datatype, vcclStream_t stream);

/* The 4-bit cache of one layer. */
typedef struct {
  void* data;
  int pages;
  int pageSize;
  int kvHeads;
  int D;
} vcclKv4_t;

/* Writes k, v [tokens, kvHeads, D] to slots (distinct where not skipped).
 * With rope (and q, qOut) the queries and keys go through vcclQkNormRope
 * first: qOut is written, and the keys are rounded to the type and stored.
 * A group of 64 channels with a NaN or an infinity, or whose extremes' sum or
 * difference is not an f32, is stored as NaN. */
vcclResult_t vcclKv4Append(const vcclKv4_t* cache, const vcclHeads_t* k, const vcclHeads_t* v, const int* slots,
                           const vcclRope_t* rope, const vcclHeads_t* q, const vcclHeads_t* qOut, int tokens,
                           vcclDataType_t datatype, vcclStream_t stream);

/* The values that the cache holds at slots; zero where a slot is skipped.
 * datatype: vcclBfloat16, vcclFloat16 or vcclFloat32. */
vcclResult_t vcclKv4Read(const vcclKv4_t* cache, const int* slots, const vcclHeads_t* k, const vcclHeads_t* v,
                         int tokens, vcclDataType_t datatype, vcclStream_t stream);

/* Causal attention of ragged query rows over the cache.  Request b owns rows
 * [qStarts[b], qStarts[b + 1]) of q and the kvLens[b] tokens of the pages in
 * table[b, :] (width columns); its last row sees all of them, the row before
 * one less, and so on.  out = softmax(scale * q k^T) v; lse (f32
 * [tokens, q heads], may be NULL) = the logarithm of the sum of exponentials.
 * A row that sees nothing is 0 with lse = -inf; one whose channels are all
 * below 2^-114 counts as zero.  Rows behind the last
 * request: 0 and -inf with zeroTail, else left as they are.  Tokens on a page
 * outside of the cache are not seen.  qStarts must not fall: the rows of
 * requests that overlap are undefined (nothing outside of out, lse and the
 * workspace is touched).  q heads a multiple of kvHeads,
 * batch <= 4096, width * pageSize <= 2^30.  workspace: vcclKv4AttentionWorkspace bytes. */
size_t vcclKv4AttentionWorkspace(int batch, int tokens, int qHeads, int kvHeads, int D);
vcclResult_t vcclKv4Attention(const vcclHeads_t* q, const vcclKv4_t* cache, const int* table, int width,
                              const int* kvLens, const int* qStarts, int batch, int tokens, float scale,
                              const vcclHeads_t* out, float* lse, int zeroTail, void* workspace,
                              vcclDataType_t datatype, vcclStream_t stream);

/* The waits inside of vcclKv4Attention are bounded.  A launch that gave one up
 * leaves its output incomplete and sets a word in host memory; the next
 * vcclKv4Attention on that device returns vcclInternalError and clears it.  A
 * program that replays a captured call makes no next call: this looks at the
 * word of the current device, with the same result (vcclSuccess where nothing
 * gave up).  It launches nothing and waits for nothing, so synchronise first. */
vcclResult_t vcclKv4AttentionStatus(void);

#ifdef __cplusplus
}
#endif

#endif /* VCCL_MODEL_H_ */
