// What the decode attentions share: the arguments and checks of a paged pool, and the launch that merges the shares of a
// sequence. Kernels: token_attention.hip (float pools), token_attention_int8.hip, token_attention_prefix.hip.
#pragma once

#include "common.hpp"

namespace amd {

constexpr float kLog2eTA = 1.4426950408889634f;
constexpr int kTaMaxSplit = 256;  // decodeMergeWideKernel holds four splits' weights per lane
constexpr int kTaGenericMaxD = 1024;  // four elements of the head row per thread

__device__ __forceinline__ int64_t ldIndex(const void* p, int64_t i, bool is64) {
  return is64 ? reinterpret_cast<const int64_t*>(p)[i] : static_cast<int64_t>(reinterpret_cast<const int32_t*>(p)[i]);
}

// Tokens of sequence b: a length outside [0, maxLen], what the table's row holds, is cut to that. All launches of a call take it from
// here: partial results are merged where they were written, and nowhere else. As two words, the second for 32-bit lengths the first
// again: a conversion in a branch on the type would wait for the length before anything else is asked for (0.3 us of the small merges).
__device__ __forceinline__ int cutLength(const void* bLen, int64_t b, bool is64, int maxLen) {
  const int* const p = static_cast<const int*>(bLen) + (b << (is64 ? 1 : 0));
  const int low = p[0], high = p[is64 ? 1 : 0];
  return high < 0 ? 0 : is64 && high != 0 ? maxLen : (int)min((unsigned)low, (unsigned)maxLen);
}
// Chunks of a sequence whose partial results are written: those that hold tokens, and the first.
__device__ __forceinline__ int chunksWritten(int len, int chunk) { return len <= 0 ? 1 : (len - 1) / chunk + 1; }

struct TaArgs {
  const void* q;
  const void* k;
  const void* v;
  const void* bLoc;
  const void* bStart;
  const void* bLen;
  bool loc64, start64, len64;
  bool generic;  // head rows the vector kernels do not take: the generic kernels run
  int64_t locRowStride;  // elements
  int64_t kSlotStride, kHeadStride, vSlotStride, vHeadStride;  // elements
  int64_t qBatchStride, qHeadStride;
  int64_t slots;
  int heads, kvHeads, d, maxLen, nsplit, chunk;
  float scaleLog2e;  // log2(e) / sqrt(d)
  const void* logits;  // two-call form: scores [heads, total_tokens], row h at logits + h * logitsHeadStride (elements)
  int64_t logitsHeadStride;
  int qGroups;  // grouped-query layouts: workgroups that share the query heads of one K/V head between them
  int batch;    // sequences (the grouped-query kernels decode a one-dimensional grid)
  const float* shared;  // decodePartials: partial results [batch, heads, nShared, 2 + d] of other tokens of the sequences, as in mergeChunks
  int nShared;
  // With a window: bLoc and maxLen are those of the tokens that are seen, the first `sinks` and the last others, right-aligned where they
  // are all there are; of a sequence that has more (up to tableLen) the first ones lie as far to the left as it is longer.
  int sinks, tableLen;
};

// max / sum of one value per thread over the workgroup of 256 (red: 4 floats of LDS; two barriers)
__device__ __forceinline__ float blockMax256(float v, float* red) {
  v = waveMax(v);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  v = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
  __syncthreads();
  return v;
}
__device__ __forceinline__ float blockSum256(float v, float* red) {
  v = waveSum(v);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  v = red[0] + red[1] + red[2] + red[3];
  __syncthreads();
  return v;
}

// Adjacent elements of a result, which may begin at any of them: one store, but of no more alignment than an element has.
template <typename V, typename T>
__device__ __forceinline__ void storeElements(T* at, const V& v) {
  __builtin_memcpy(at, &v, sizeof(V));
}

// x - ref where x is a product that is rounded before: a multiply-add (which the compiler makes of the two by itself) keeps in the
// difference what ref, another such product, lost in rounding.
__device__ __forceinline__ float behindRounded(float x, float ref) {
#pragma clang fp contract(off)
  return x - ref;
}

// ---------------------------------------------------------------- host side --
struct TaViews {
  TensorView q, k, v, loc, start, len;
};

// q, the slot table, the starts and the lengths alone: checked, and in `a` (the rest of it zero).
diopiError_t tableArgs(const TaViews& t, int maxLen, TaArgs* a);
// q, k, v (those needed), the slot table, the starts and the lengths: checked, and their strides and types in `a`.
diopiError_t fillArgs(const TaViews& t, bool needK, bool needV, int maxLen, TaArgs* a);

// out[b, h, :] (dense, `dtype`) from the partial results [batch, heads, nsplit, 2 + d] of chunks of `a.chunk` tokens: maximum (in
// units of log2), sum and weighted sum of V, chunk i written where i = 0 or a sequence has more than i * chunk tokens.
diopiError_t mergeChunks(hipStream_t stream, diopiDtype_t dtype, void* out, const float* partial, const TaArgs& a, int64_t batch);

// diopiTokenDecodeAttentionInference's kernels (not for generic arguments) behind other tokens, whose partial results are in a.shared.
// Sequences of one chunk: the result, in `out` (*keep is empty). Longer ones, or where a.shared has too many shares for that: partial results
// of at least two chunks, which mergeChunks could merge, in workspace of the context.
struct TaPartials {
  const float* partial;
  int nsplit, chunk;
  float raise;  // sums are against the maximum less this (in units of log2)
};
diopiError_t decodePartials(diopiContextHandle_t ctx, hipStream_t stream, const TaArgs& a, diopiDtype_t dtype, int maxInputLen, void* out, TaPartials* keep);

// diopiTokenDecodeAttentionInference's kernels (not for generic arguments) over the last `window` tokens of each sequence and its first
// `sinks`, window + sinks < a.maxLen. (64 x (512 .. 6000) tokens, window 2048, 32 heads of 128 bf16 317 us, 6.1 TB/s; 48 x (100 .. 12000), window 2048 and 4
// first ones, 32 heads on 8 fp16 73 us, 5.1 TB/s; the 64 in fp32 610 us, 6.1 TB/s)
diopiError_t decodeWindow(diopiContextHandle_t ctx, hipStream_t stream, TaArgs a, diopiDtype_t dtype, int window, int sinks, void* out);

// As decodePartials, for rows of any kind and for int8 pools: partial results of the first `walked` tokens in `loc` and the own ones behind
// them, of at least one chunk; if nothing else is to be merged (alone) and there is one chunk, the result (own->nsplit is 0 then).
struct TaAnyArgs {
  TaArgs a;
  const void* loc;  // slots of shared tokens
  bool locIs64;
  int walked;
  const float* kScale;  // null: the pool is of q's type
  const float* vScale;
  int64_t kScaleSlot, kScaleHead, vScaleSlot, vScaleHead;
  int chunk, split;  // (set by walkAny)
};
diopiError_t walkAny(diopiContextHandle_t ctx, hipStream_t stream, TaAnyArgs x, diopiDtype_t dtype, void* out, bool alone, TaPartials* own);

// out from the partial results of nShared chunks of tokens that all sequences have and `own` of what comes behind (with `walked` of the
// shared tokens in front).
diopiError_t mergeShares(hipStream_t stream, const TaArgs& a, diopiDtype_t dtype, void* out, const float* shared, int nShared, const TaPartials& own, int walked);

}  // namespace amd
