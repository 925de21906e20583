// Attention of new tokens over a paged pool: arguments, what a token sees, and how a launch's workgroups find their work.
// Kernels: paged_attention.hip (any rows, entry points), paged_attention_mfma.hip.
#pragma once

#include "token_attention.hpp"

namespace amd {

struct PaArgs {
  const void* q;
  const void* k;
  const void* v;
  void* out;
  const void* bLoc;
  const void* bStart;
  const void* bNew;  // null: one new token for each sequence, in row b of q
  const void* bLen;
  bool loc64, start64, new64, len64;
  int64_t locRowStride;                                     // elements
  int64_t kSlotStride, kHeadStride, vSlotStride, vHeadStride;  // elements
  int64_t qTok, qHead, oTok, oHead;                         // elements
  int64_t slots, rows;                                      // of the pool; of q
  int heads, kvHeads, d, batch, maxNew, maxLen;
  int window, sinks;  // a token at position p sees j <= p with j > p - window or j < sinks (window: maxLen or more where there is none)
  float scaleLog2e;   // log2(e) / sqrt(d)
};

#if defined(__HIPCC__)

// The new tokens of a sequence that have a row in q, [first, end), and the position of token 0.
struct PaSequence {
  int64_t start;  // row of token 0
  int first, end, origin;
};
__device__ __forceinline__ PaSequence paSequence(const PaArgs& a, int b) {
  PaSequence s;
  const int len = cutLength(a.bLen, b, a.len64, a.maxLen);
  const int n = a.bNew == nullptr ? 1 : cutLength(a.bNew, b, a.new64, a.maxNew);
  s.start = a.bNew == nullptr ? b : ldIndex(a.bStart, b, a.start64);
  s.origin = len - n;
  // rows outside q are left out (bounds first: a start may be any number)
  s.first = s.start >= 0 ? 0 : (int)min((int64_t)n, s.start < -(int64_t)n ? (int64_t)n : -s.start);
  s.end = s.start >= a.rows ? s.first : (int)min((int64_t)n, a.rows - max(s.start, -(int64_t)n));
  s.end = max(s.end, s.first);
  return s;
}

// Where in the list of all sequences' pieces, count(sequence) of each, piece `u` lies: its sequence (-1: behind the last) and its number
// there. total: all of them. Every lane of the wave takes part, and all get the same.
struct PaPlace {
  int b, at;
  int64_t total;
};
template <typename F>
__device__ __forceinline__ PaPlace paFind(const PaArgs& a, int64_t u, F&& count) {
  const int lane = threadIdx.x & 63;
  PaPlace p{-1, 0, 0};
  for (int b0 = 0; b0 < a.batch; b0 += 64) {
    const int mine = b0 + lane < a.batch ? count(paSequence(a, b0 + lane)) : 0;
    int upTo = mine;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
      const int below = __shfl_up(upTo, off, 64);
      if (lane >= off) upTo += below;
    }
    const uint64_t behind = __builtin_amdgcn_ballot_w64(p.total + upTo > u);
    if (p.b < 0 && behind != 0) {
      const int l = __builtin_ctzll(behind);
      p.b = b0 + l;
      p.at = (int)(u - p.total) - (__builtin_amdgcn_readlane(upTo, l) - __builtin_amdgcn_readlane(mine, l));
    }
    p.total += __builtin_amdgcn_readlane(upTo, 63);
  }
  return p;
}

#endif

// Attention over rows of any size and layout, q and pool of one type.
diopiError_t pagedAttentionAny(hipStream_t stream, const PaArgs& a, diopiDtype_t dtype);

}  // namespace amd
