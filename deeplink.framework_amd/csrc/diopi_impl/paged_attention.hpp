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
  int group;          // query heads to a K/V head
  uint32_t perGroup;  // ceil(2^32 / group): see paOfGroup
};

#if defined(__HIPCC__)

// Index i of a tensor of 32 or 64-bit ones, as two words to be put together where it is used (the second for 32-bit ones the first again): a
// conversion in a branch on the type would wait for it, and for all loads before it, at once (2.1 instead of 1.4 us for a tile of
// pagedTileBlock, whose copies were on their way).
__device__ __forceinline__ int2 paAsk(const void* p, int64_t i, bool is64) {
  const int* const at = static_cast<const int*>(p) + (i << (is64 ? 1 : 0));
  return int2{at[0], at[is64 ? 1 : 0]};
}
__device__ __forceinline__ int64_t paIndex(int2 v, bool is64) { return is64 ? (int64_t)((uint64_t)(uint32_t)v.y << 32 | (uint32_t)v.x) : (int64_t)v.x; }

// The new tokens of a sequence that have a row in q, [first, end), and the position of token 0.
struct PaSequence {
  int64_t start;  // row of token 0
  int first, end, origin, len;
};
__device__ __forceinline__ PaSequence paSequence(const PaArgs& a, int b) {
  PaSequence s;
  int2 start{b, 0};
  if (a.bNew != nullptr) start = paAsk(a.bStart, b, a.start64);
  const int len = cutLength(a.bLen, b, a.len64, a.maxLen);
  const int n = a.bNew == nullptr ? 1 : cutLength(a.bNew, b, a.new64, a.maxNew);
  s.start = a.bNew == nullptr ? b : paIndex(start, a.start64);
  s.origin = len - n, s.len = len;
  // rows outside q are left out (bounds first: a start may be any number)
  s.first = s.start >= 0 ? 0 : (int)min((int64_t)n, s.start < -(int64_t)n ? (int64_t)n : -s.start);
  s.end = s.start >= a.rows ? s.first : (int)min((int64_t)n, a.rows - max(s.start, -(int64_t)n));
  s.end = max(s.end, s.first);
  return s;
}

// Where in the list of all sequences' pieces, count(sequence) of each, piece `u` lies: its sequence (b = -1: behind the last) and its
// number there. total: all of them. Every lane of the wave takes part, and all get the same.
struct PaPlace {
  int b, at;
  int64_t total;
  PaSequence s;
};
template <typename F>
__device__ __forceinline__ PaPlace paFind(const PaArgs& a, int64_t u, F&& count) {
  const int lane = threadIdx.x & 63;
  PaPlace p;
  p.b = -1, p.at = 0, p.total = 0;
  for (int b0 = 0; b0 < a.batch; b0 += 64) {
    const PaSequence s = paSequence(a, min(b0 + lane, a.batch - 1));
    const int mine = b0 + lane < a.batch ? count(s) : 0;
    int upTo = mine;
    if (a.batch > 1) {
#pragma unroll
      for (int off = 1; off < 64; off <<= 1) {
        const int below = __shfl_up(upTo, off, 64);
        if (lane >= off) upTo += below;
      }
    }
    const uint64_t behind = __builtin_amdgcn_ballot_w64(b0 + lane < a.batch && p.total + upTo > u);
    if (p.b < 0 && behind != 0) {
      const int l = __builtin_ctzll(behind);
      auto of = [&](int v) { return __builtin_amdgcn_readlane(v, l); };
      p.b = b0 + l;
      p.at = (int)(u - p.total) - (of(upTo) - of(mine));
      p.s.start = (int64_t)((uint64_t)(uint32_t)of((int)(s.start >> 32)) << 32 | (uint32_t)of((int)s.start));
      p.s.first = of(s.first), p.s.end = of(s.end), p.s.origin = of(s.origin), p.s.len = of(s.len);
    }
    p.total += __builtin_amdgcn_readlane(upTo, min(63, a.batch - 1 - b0));
  }
  return p;
}

// n / group, for n * group below 2^32: the product with the rounded-up reciprocal is too large by less than n / 2^32, which is below 1 / group.
__device__ __forceinline__ int paOfGroup(const PaArgs& a, int n) { return a.group == 1 ? n : (int)__umulhi((uint32_t)n, a.perGroup); }

// The tokens that one at position p sees: [0, head) and [low, p].
__device__ __forceinline__ void paSeen(const PaArgs& a, int p, int* head, int* low) {
  *low = max(0, p - a.window + 1);
  *head = max(0, min(a.sinks, min(*low, p + 1)));
}

// A wave's part of the attention of one (new token, head), any layout: the tokens [first0, first1) and [next0, next1) of the sequence,
// 64 at a time from the `offset`th on and every `step`th 64 of them. A row is spread over the lanes (element lane + 64 j), UNR rows are
// asked for at once; slots outside the pool are skipped, never dereferenced. m: the largest score in units of log2, l and acc: sums of
// the weights against it, and of V.
template <typename T, int J, int UNR>
struct PaColumn {
  float m = -INFINITY, l = 0.f, acc[J];
  __device__ __forceinline__ void walk(const PaArgs& a, const T* q, int kvh, int64_t locBase, int first0, int first1, int next0, int next1, int offset, int step) {
    const int lane = threadIdx.x & 63, head = max(0, first1 - first0), n = head + max(0, next1 - next0);
    const T* kHead = reinterpret_cast<const T*>(a.k) + kvh * a.kHeadStride;
    const T* vHead = reinterpret_cast<const T*>(a.v) + kvh * a.vHeadStride;
    int at[J];  // the lane's elements of a row; past its end the first one, which q's zero leaves out
    float qf[J];
#pragma unroll
    for (int j = 0; j < J; ++j) {
      const int e = lane + 64 * j;
      at[j] = e < a.d ? e : 0;
      qf[j] = e < a.d ? static_cast<float>(q[e]) * a.scaleLog2e : 0.f;
      acc[j] = 0.f;
    }
    for (int t0 = offset; t0 < n; t0 += step) {
      const int i0 = min(t0 + lane, n - 1), cnt = min(64, n - t0);
      int64_t mine = ldIndex(a.bLoc, locBase + (i0 < head ? first0 + i0 : next0 + (i0 - head)), a.loc64);
      if (mine < 0 || mine >= a.slots) mine = -1;
      for (int i = 0; i < cnt; i += UNR) {
        float k[UNR][J], v[UNR][J], sc[UNR], mt = m;
        bool counts[UNR];
#pragma unroll
        for (int w = 0; w < UNR; ++w) {
          const int from = min(i + w, cnt - 1);
          const int64_t slot = (int64_t)((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(mine >> 32), from) << 32 | (uint32_t)__builtin_amdgcn_readlane((int)mine, from));
          counts[w] = i + w < cnt && slot >= 0;
          const T* kRow = kHead + max(slot, (int64_t)0) * a.kSlotStride;
          const T* vRow = vHead + max(slot, (int64_t)0) * a.vSlotStride;
#pragma unroll
          for (int j = 0; j < J; ++j) k[w][j] = static_cast<float>(kRow[at[j]]), v[w][j] = static_cast<float>(vRow[at[j]]);
        }
#pragma unroll
        for (int w = 0; w < UNR; ++w) {
          float dot = 0.f;
#pragma unroll
          for (int j = 0; j < J; ++j) dot += lane + 64 * j < a.d ? qf[j] * k[w][j] : 0.f;
          sc[w] = waveSum(dot);
          if (!counts[w]) sc[w] = -INFINITY;
          mt = fmaxf(mt, sc[w]);
        }
        const float ref = mt == -INFINITY ? 0.f : mt, corr = m == -INFINITY ? 1.f : exp2f(m - ref);  // (no maximum yet: the sums are 0, or NaN)
        m = mt, l *= corr;
#pragma unroll
        for (int j = 0; j < J; ++j) acc[j] *= corr;
#pragma unroll
        for (int w = 0; w < UNR; ++w) {
          if (!counts[w]) continue;
          const float e = exp2f(behindRounded(sc[w], ref));
          l += e;
#pragma unroll
          for (int j = 0; j < J; ++j) acc[j] += e * v[w][j];
        }
      }
    }
    if (l != l && m == -INFINITY) m = 0.f;  // scores that are not numbers alone: as a maximum of minus infinity they would be left out
  }
};

#endif

// Attention over rows of any size and layout, q and pool of one type.
diopiError_t pagedAttentionAny(hipStream_t stream, const PaArgs& a, diopiDtype_t dtype);

// Attention on the matrix pipe: whether it takes these rows, and its launches.
bool pagedAttentionTiles(const PaArgs& a, diopiDtype_t dtype);
diopiError_t pagedAttentionMfma(diopiContextHandle_t ctx, hipStream_t stream, const PaArgs& a, diopiDtype_t dtype);

}  // namespace amd
