// The int8 KV cache for gfx950: rows quantised as they are written into the pool, and read back.
//
//   k, v [tokens, kv_heads, d]          new rows (fp16, bf16 or fp32)
//   pool [slots, kv_heads, d] int8, scale [slots, kv_heads] fp32
//
// A row (one token, one head) x is kept as whole numbers q and a scale s:
//   s = max |x| / 127 rounded to fp32,  q = the whole number nearest to x / s, ties to the even one
// so q lies in [-127, 127] (it is cut to that where s has lost its last places below 2^-126). q is that of the EXACT quotient: a
// quotient rounded to fp32 falls on a half for one element in 10^5 that does not, and which neighbour it goes to would depend on
// how the division is done. Rows of zeros have s = 0. A row that holds an infinity or NaN has s = NaN and q = 0: all of it reads
// back as NaN, none of it as a plausible number. Read back: q * s rounded to fp32, and once more to a 16-bit type.
//
// Both are bound by memory: a 16-bit row of 128 moves 256 + 132 bytes. Reading 15001 rows of 40 heads back takes 84 us, 5.6 TB/s.
// Writing 8192 of 32 takes 45 us, 4.5 TB/s, about 6 of them to find repeated slots; its arithmetic, 9 instructions an element, is nearly as long.
//   * a row is spread over LPR lanes of 8 elements each (16 bytes of a 16-bit type in, 8 bytes out), so that the largest
//     magnitude is a few lane permutations; a lane asks for kKvRows rows before it works on the first;
//   * quotients go through the reciprocal and are rounded by an addition; only where a remainder could decide otherwise is it
//     computed (see below). Two divisions to a row and a check of each element's remainder took 95 us where this takes 45;
//   * K and V are halves of the grid: the choice by an index per lane kept their addresses out of scalar registers (105 us
//     became 189 us for the read above, as it was then).
// The last of several tokens with one destination is what the slot holds, as a loop over the tokens would leave it (a row and its
// scale must not come from two tokens). A workgroup looks through the destinations behind its own while its rows are on their
// way; above kKvScanTokens tokens two launches of their own find the last of each first.
#include <algorithm>

#include "common.hpp"

namespace amd {

constexpr int kKvThreads = 256;
constexpr int kKvRows = 4;               // rows that a lane group has in flight
constexpr int kKvTokensPerWg = 8;        // most tokens of a workgroup that writes
// Workgroups look for later tokens with the same slot themselves up to this many tokens: 4096 tokens of 8 heads are written in 11.1 us so,
// 4097 in 14.2 with the two launches before; of 32 heads in 27.7 and 26.6.
constexpr int64_t kKvScanTokens = 4096;

struct KvInt8Pool {
  void* x;           // rows in the activations' type: read (write into the pool) or written (read back)
  int8_t* pool;
  float* scale;
  int64_t xToken, xHead;                     // strides in elements
  int64_t poolSlot, poolHead, scaleSlot, scaleHead;
};
struct KvInt8Args {
  KvInt8Pool pool[2];
  const void* loc;
  bool loc64;
  int64_t tokens, slots;
  int heads, d;
  float perHeads;    // 1 / heads
  int tokensPerWg;
  const int* last;   // the last token of each slot (null: the workgroups that write look for themselves)
};

__device__ __forceinline__ int64_t kvSlot(const KvInt8Args& a, int64_t t) {
  return a.loc64 ? static_cast<const int64_t*>(a.loc)[t] : static_cast<int64_t>(static_cast<const int32_t*>(a.loc)[t]);
}
// A destination counted from the end if negative; -1 outside the pool (dropped, never written).
__device__ __forceinline__ int kvDestination(const KvInt8Args& a, int64_t slot) {
  if (slot < 0) slot += a.slots;
  return slot >= 0 && slot < a.slots ? (int)slot : -1;
}
// Row i of a workgroup's (token, head) pairs, heads fastest: its token. i + 1/2 over the heads is at least half a head away from a
// whole number, and the product is off by less for i up to 2^21.
__device__ __forceinline__ int kvTokenOf(const KvInt8Args& a, int i) { return (int)(((float)i + 0.5f) * a.perHeads); }

// What the magnitudes of a row and their largest (as bits: an infinity is above every number, NaN above that) make of it.
struct KvScale {
  float scale;    // what is stored
  float up;       // rows of tiny numbers are lifted by 2^64 first, so that 1 / scale is finite
  float s, inv, half;
  bool special;   // tiny, or not finite
  __device__ __forceinline__ explicit KvScale(uint32_t bits) {
    const float most = __uint_as_float(bits);
    const bool finite = bits < 0x7f800000u;
    special = !finite || (most < 0x1p-60f && bits != 0);
    // most / 127, rounded once: the quotient by the rounded reciprocal, corrected by its remainder, which the fused multiply-add gives
    // exactly (P. Markstein, 1990; not where results lose places below 2^-126)
    constexpr float kPer127 = 1.f / 127.f;
    const float rough = most * kPer127;
    scale = special ? most / 127.f : fmaf(fmaf(-127.f, rough, most), kPer127, rough);
    if (!finite) scale = __uint_as_float(0x7fc00000u);
    up = most < 0x1p-60f ? 0x1p64f : 1.f;
    s = scale * up;
    inv = finite && s > 0.f ? __builtin_amdgcn_rcpf(s) : 0.f;  // (off by 2^-23 at most)
    half = 0.5f * s;
  }
  // The whole number nearest to x / scale. x * inv is off by less than 2^-14, so its nearest whole number is that or a
  // neighbour of it, and the remainder says which: x - q s is a multiple of the smaller of the last places of x and s and at most
  // a little more than s / 2, so it fits 24 bits and the fused multiply-add gives it exactly.
  __device__ __forceinline__ int nearest(float x) const {
    x *= up;
    float q = __builtin_rintf(x * inv);
    const float r = fmaf(-q, s, x), d = fabsf(r);
    const int odd = static_cast<int>(q) & 1;
    if (d > half || (d == half && odd)) q += r > 0.f ? 1.f : -1.f;
    // (a scale that is a handful of the smallest numbers may be a third too small)
    return inv > 0.f ? min(max(static_cast<int>(q), -127), 127) : 0;
  }
};

// The largest of one value per lane over the LPR adjacent lanes that share a row.
template <int LPR>
__device__ __forceinline__ uint32_t rowMost(uint32_t v) {
  auto other = [&](auto ctrl) { return (uint32_t)__builtin_amdgcn_update_dpp((int)v, (int)v, decltype(ctrl)::value, 0xf, 0xf, false); };
  v = max(v, other(std::integral_constant<int, kDppQuadSwap1>{}));
  v = max(v, other(std::integral_constant<int, kDppQuadSwap2>{}));
  v = max(v, other(std::integral_constant<int, kDppHalfMirror>{}));
  if (LPR >= 16) v = max(v, other(std::integral_constant<int, kDppMirror>{}));
  if (LPR >= 32) v = max(v, (uint32_t)__shfl_xor((int)v, 16, 64));
  return v;
}

template <typename T>
struct KvPiece {  // 8 elements
  typename Vec16<T>::type v[8 / Vec16<T>::N];
  // the largest magnitude as the bits of an fp32 number, an infinity above every number and NaN above that (16-bit types: pairs at once, and
  // the largest is converted)
  __device__ __forceinline__ uint32_t most() const {
    if constexpr (sizeof(T) == 4) {
      uint32_t m = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint((*this)[i]) & 0x7fffffffu);
      return m;
    } else {
      typedef uint16_t Pair __attribute__((ext_vector_type(2)));
      const u32x4 w = __builtin_bit_cast(u32x4, v[0]) & 0x7fff7fffu;
      auto larger = [](uint32_t x, uint32_t y) {
        return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(Pair, x), __builtin_bit_cast(Pair, y)));
      };
      const uint32_t m = larger(larger(w[0], w[1]), larger(w[2], w[3]));
      const uint16_t top = max((uint16_t)m, (uint16_t)(m >> 16));
      return __float_as_uint(static_cast<float>(__builtin_bit_cast(T, top)));
    }
  }
  __device__ __forceinline__ float operator[](int i) const { return static_cast<float>(v[i / Vec16<T>::N][i % Vec16<T>::N]); }
};

struct KvSlot {  // where a token's rows and scales begin in the pools: looked up once per token
  int64_t pool, scale;
  int slot;  // -1: none
  __device__ __forceinline__ KvSlot() {}
  __device__ __forceinline__ KvSlot(const KvInt8Pool& o, int slot) : pool(max(slot, 0) * o.poolSlot), scale(max(slot, 0) * o.scaleSlot), slot(slot) {}
};

// The slots that a workgroup which writes asks for first: those of its own tokens (in lane i of every wave that of token i) and, where
// it looks for repeated ones itself (SCAN), of the kKvBatch * kKvThreads tokens behind them. As two words, the second for 32-bit slots
// the first again: a branch on the type would wait for one load before it asks for the next.
constexpr int kKvBatch = 8;
template <bool SCAN>
struct KvAsked {
  int2 own, behind[SCAN ? kKvBatch : 1];
};
__device__ __forceinline__ int2 kvAsk(const KvInt8Args& a, int64_t t) {
  const int* p = static_cast<const int*>(a.loc) + (t << (a.loc64 ? 1 : 0));
  return int2{p[0], p[a.loc64 ? 1 : 0]};
}
__device__ __forceinline__ int kvDestination(const KvInt8Args& a, int2 slot) {
  return kvDestination(a, a.loc64 ? (int64_t)((uint64_t)(uint32_t)slot.y << 32 | (uint32_t)slot.x) : (int64_t)slot.x);
}
template <bool SCAN>
__device__ __forceinline__ KvAsked<SCAN> kvAskFirst(const KvInt8Args& a, int64_t t0, int n) {
  KvAsked<SCAN> asked;
  asked.own = kvAsk(a, t0 + min((int)(threadIdx.x & 63), n - 1));
  if constexpr (SCAN) {
#pragma unroll
    for (int k = 0; k < kKvBatch; ++k) asked.behind[k] = kvAsk(a, min(t0 + n + threadIdx.x + k * kKvThreads, a.tokens - 1));
  }
  __builtin_amdgcn_sched_barrier(0);  // (ahead of the rows: loads return in order, and the search goes on while those are on their way)
  return asked;
}

// Whether a later token has the slot of one of the MOST tokens [t0, t0 + n) of the workgroup, as bits. `mine`: in lane i of every
// wave the slot of token t0 + i, -1 where there is none.
template <int MOST>
__device__ __forceinline__ unsigned kvLater(const KvInt8Args& a, int64_t t0, int n, int mine, const int2 (&first)[kKvBatch]) {
  int slot[MOST];
  uint64_t same[MOST];
  unsigned later = 0;
#pragma unroll
  for (int i = 0; i < MOST; ++i) {
    slot[i] = __builtin_amdgcn_readlane(mine, i);  // (in a scalar register: a comparison each, and nothing else)
    same[i] = __builtin_amdgcn_ballot_w64(mine == slot[i]) >> (i + 1);  // among the workgroup's own
  }
  auto compare = [&](int2 asked) {
    const int s = kvDestination(a, asked);
#pragma unroll
    for (int i = 0; i < MOST; ++i) same[i] |= __builtin_amdgcn_ballot_w64(s == slot[i]);
  };
  const int64_t begin = t0 + n;
#pragma unroll
  for (int k = 0; k < kKvBatch; ++k) {
    if (begin + k * kKvThreads >= a.tokens) break;
    compare(first[k]);  // (past the last token: that again)
  }
  for (int64_t j0 = begin + kKvThreads * kKvBatch; j0 < a.tokens; j0 += kKvThreads * kKvBatch) {
    int2 at[kKvBatch];
#pragma unroll
    for (int k = 0; k < kKvBatch; ++k) at[k] = kvAsk(a, min(j0 + threadIdx.x + k * kKvThreads, a.tokens - 1));
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int k = 0; k < kKvBatch; ++k) compare(at[k]);
  }
#pragma unroll
  for (int i = 0; i < MOST; ++i) later |= same[i] != 0 ? 1u << i : 0u;
  return later;
}

// The slots of the workgroup's tokens [t0, t0 + n), -1 for those that are not written: no destination, or a later token has the
// same. (One barrier; every thread of the workgroup takes part.)
template <bool SCAN>
__device__ __forceinline__ void kvDestinations(const KvInt8Args& a, int64_t t0, int n, const KvAsked<SCAN>& asked, KvSlot (&slots)[kKvTokensPerWg],
                                               unsigned (&later)[kKvThreads / 64]) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int mine = lane < n ? kvDestination(a, asked.own) : -1;
  unsigned found = 0;
  if constexpr (SCAN) {
    found = n <= 2 ? kvLater<2>(a, t0, n, mine, asked.behind) : kvLater<kKvTokensPerWg>(a, t0, n, mine, asked.behind);
  } else {
    if (mine >= 0 && a.last[mine] != (int)(t0 + lane)) mine = -1;
  }
  if (lane == 0) later[wave] = found;
  if (wave == 0 && lane < kKvTokensPerWg) slots[lane] = KvSlot(a.pool[blockIdx.y], mine);
  __syncthreads();
}

// grid: (workgroups of tokensPerWg tokens, K or V). Rows of a workgroup: (token, head), head fastest.
template <typename T, int LPR, bool SCAN>
__global__ __launch_bounds__(kKvThreads) void kvInt8WriteKernel(KvInt8Args a) {
  constexpr int kGroups = kKvThreads / LPR;
  __shared__ unsigned later[kKvThreads / 64];
  __shared__ KvSlot slots[kKvTokensPerWg];
  const int64_t t0 = (int64_t)blockIdx.x * a.tokensPerWg;
  const int n = (int)min((int64_t)a.tokensPerWg, a.tokens - t0);
  const int sub = threadIdx.x % LPR, group = threadIdx.x / LPR;
  const KvInt8Pool& o = a.pool[blockIdx.y];
  const int rows = n * a.heads, e = sub * 8;
  const bool live = e < a.d;
  const T* const from = static_cast<const T*>(o.x) + t0 * o.xToken;
  KvPiece<T> x[kKvRows];
  int token[kKvRows], head[kKvRows];
  auto load = [&](int r0) {
#pragma unroll
    for (int u = 0; u < kKvRows; ++u) {
      const int r = min(r0 + u * kGroups, rows - 1);
      token[u] = kvTokenOf(a, r), head[u] = r - token[u] * a.heads;
      const T* src = from + (__umul24(token[u], (unsigned)o.xToken) + __umul24(head[u], (unsigned)o.xHead) + (live ? e : 0));
#pragma unroll
      for (int c = 0; c < 8 / Vec16<T>::N; ++c) x[u].v[c] = __builtin_nontemporal_load(reinterpret_cast<const typename Vec16<T>::type*>(src) + c);
    }
  };
  const KvAsked<SCAN> asked = kvAskFirst<SCAN>(a, t0, n);
  load(group);
  kvDestinations<SCAN>(a, t0, n, asked, slots, later);
  const unsigned dead = later[0] | later[1] | later[2] | later[3];
  for (int r0 = group; r0 < rows; r0 += kKvRows * kGroups) {
    if (r0 != group) load(r0);
#pragma unroll
    for (int u = 0; u < kKvRows; ++u) {
      const KvScale s(rowMost<LPR>(live ? x[u].most() : 0));
      // x / s by the reciprocal, rounded by adding 3 * 2^22: the last byte of the sum is the whole number. It is the nearest one
      // unless the quotient is within 2^-15 (twice what 127 times the reciprocal can be off by) of a half; such rows, tiny ones
      // and those that are not finite go element by element
      constexpr float kWhole = 12582912.f;
      float t[8], off = 0.f;
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        t[k] = fmaf(x[u][k], s.inv, kWhole);
        off = fmaxf(off, fabsf(fmaf(x[u][k], s.inv, kWhole - t[k])));
      }
      u32x2 q;
#pragma unroll
      for (int w = 0; w < 2; ++w) {
        const uint32_t low = __builtin_amdgcn_perm(__float_as_uint(t[4 * w + 1]), __float_as_uint(t[4 * w]), 0x0c0c0400u);
        const uint32_t high = __builtin_amdgcn_perm(__float_as_uint(t[4 * w + 3]), __float_as_uint(t[4 * w + 2]), 0x0c0c0400u);
        q[w] = low | high << 16;
      }
      if (__builtin_amdgcn_ballot_w64(!(off < 0.49996f) || s.special) != 0) {
        q = u32x2{0, 0};
#pragma unroll
        for (int k = 0; k < 8; ++k) q[k / 4] |= (uint32_t)(s.nearest(x[u][k]) & 255) << (8 * (k % 4));
      }
      const KvSlot to = slots[token[u]];
      if (r0 + u * kGroups >= rows || to.slot < 0 || (dead >> token[u] & 1)) continue;
      if (live) *reinterpret_cast<u32x2*>(o.pool + (to.pool + __umul24(head[u], (unsigned)o.poolHead) + e)) = q;
      if (sub == 0) o.scale[to.scale + __umul24(head[u], (unsigned)o.scaleHead)] = s.scale;
    }
  }
}

// Any head size and alignment: a wave per row.
template <typename T, bool SCAN>
__global__ __launch_bounds__(kKvThreads) void kvInt8WriteAnyKernel(KvInt8Args a) {
  __shared__ unsigned later[kKvThreads / 64];
  __shared__ KvSlot slots[kKvTokensPerWg];
  const int64_t t0 = (int64_t)blockIdx.x * a.tokensPerWg;
  const int n = (int)min((int64_t)a.tokensPerWg, a.tokens - t0);
  kvDestinations<SCAN>(a, t0, n, kvAskFirst<SCAN>(a, t0, n), slots, later);
  const unsigned dead = later[0] | later[1] | later[2] | later[3];
  const int lane = threadIdx.x & 63, rows = n * a.heads;
  const KvInt8Pool& o = a.pool[blockIdx.y];
  for (int r = threadIdx.x / 64; r < rows; r += kKvThreads / 64) {
    const int t = r / a.heads, h = r - t * a.heads;
    const int slot = slots[t].slot;
    if (slot < 0 || (dead >> t & 1)) continue;
    const T* src = static_cast<const T*>(o.x) + (t0 + t) * o.xToken + h * o.xHead;
    uint32_t most = 0;
    for (int e = lane; e < a.d; e += 64) most = max(most, __float_as_uint(static_cast<float>(src[e])) & 0x7fffffffu);
    most = rowMost<32>(most);
    const KvScale s(max(most, (uint32_t)__shfl_xor((int)most, 32, 64)));
    int8_t* dst = o.pool + slot * o.poolSlot + h * o.poolHead;
    for (int e = lane; e < a.d; e += 64) dst[e] = static_cast<int8_t>(s.nearest(static_cast<float>(src[e])));
    if (lane == 0) o.scale[slot * o.scaleSlot + h * o.scaleHead] = s.scale;
  }
}

// last[slot]: the last token whose destination it is, in two launches. Entries need no first value: every token writes its own to
// begin with (one of a slot's tokens stays there), and then the largest replaces it.
template <bool FIRST>
__global__ __launch_bounds__(kKvThreads) void kvInt8LastKernel(KvInt8Args a, int* last) {
  const int64_t t = (int64_t)blockIdx.x * kKvThreads + threadIdx.x;
  if (t >= a.tokens) return;
  const int s = kvDestination(a, kvSlot(a, t));
  if (s < 0) return;
  if (FIRST) last[s] = (int)t;
  else atomicMax(&last[s], (int)t);
}

// grid: (workgroups of tokensPerWg rows of `loc`, K or V)
template <typename T, int LPR>
__global__ __launch_bounds__(kKvThreads) void kvInt8ReadKernel(KvInt8Args a) {
  constexpr int kGroups = kKvThreads / LPR;
  __shared__ int slots[kKvTokensPerWg];  // -1: outside the pool
  const int64_t t0 = (int64_t)blockIdx.x * a.tokensPerWg;
  const int n = (int)min((int64_t)a.tokensPerWg, a.tokens - t0);
  if ((int)threadIdx.x < n) {
    const int64_t slot = kvSlot(a, t0 + threadIdx.x);
    slots[threadIdx.x] = slot >= 0 && slot < a.slots ? (int)slot : -1;
  }
  __syncthreads();
  const int sub = threadIdx.x % LPR, group = threadIdx.x / LPR;
  const KvInt8Pool& o = a.pool[blockIdx.y];
  const int rows = n * a.heads, e = sub * 8;
  if (e >= a.d) return;
  T* const x0 = static_cast<T*>(o.x) + t0 * o.xToken;
  for (int r0 = group; r0 < rows; r0 += kKvRows * kGroups) {
    u32x2 q[kKvRows];
    float s[kKvRows];
    unsigned to[kKvRows];
#pragma unroll
    for (int u = 0; u < kKvRows; ++u) {
      const int r = min(r0 + u * kGroups, rows - 1), t = kvTokenOf(a, r), h = r - t * a.heads;
      to[u] = __umul24(t, (unsigned)o.xToken) + __umul24(h, (unsigned)o.xHead) + e;
      const int slot = slots[t];
      q[u] = u32x2{0, 0}, s[u] = 0.f;
      if (slot >= 0) {  // outside the pool: zeros, nothing is read
        q[u] = __builtin_nontemporal_load(reinterpret_cast<const u32x2*>(o.pool + (slot * o.poolSlot + __umul24(h, (unsigned)o.poolHead) + e)));
        s[u] = o.scale[slot * o.scaleSlot + __umul24(h, (unsigned)o.scaleHead)];
      }
    }
#pragma unroll
    for (int u = 0; u < kKvRows; ++u) {
      if (r0 + u * kGroups >= rows) continue;
      KvPiece<T> x;
#pragma unroll
      for (int k = 0; k < 8; ++k)
        x.v[k / Vec16<T>::N][k % Vec16<T>::N] = static_cast<T>(static_cast<float>((int)(q[u][k / 4] << (24 - 8 * (k % 4))) >> 24) * s[u]);
      T* dst = x0 + to[u];
#pragma unroll
      for (int c = 0; c < 8 / Vec16<T>::N; ++c) __builtin_nontemporal_store(x.v[c], reinterpret_cast<typename Vec16<T>::type*>(dst) + c);
    }
  }
}

template <typename T>
__global__ __launch_bounds__(kKvThreads) void kvInt8ReadAnyKernel(KvInt8Args a) {
  const int64_t t0 = (int64_t)blockIdx.x * a.tokensPerWg;
  const int n = (int)min((int64_t)a.tokensPerWg, a.tokens - t0);
  const int lane = threadIdx.x & 63, rows = n * a.heads;
  const KvInt8Pool& o = a.pool[blockIdx.y];
  for (int r = threadIdx.x / 64; r < rows; r += kKvThreads / 64) {
    const int t = r / a.heads, h = r - t * a.heads;
    const int64_t slot = kvSlot(a, t0 + t);
    const bool in = slot >= 0 && slot < a.slots;
    const float s = in ? o.scale[slot * o.scaleSlot + h * o.scaleHead] : 0.f;
    T* dst = static_cast<T*>(o.x) + (t0 + t) * o.xToken + h * o.xHead;
    for (int e = lane; e < a.d; e += 64) dst[e] = static_cast<T>(in ? static_cast<float>(o.pool[slot * o.poolSlot + h * o.poolHead + e]) * s : 0.f);
  }
}

// ---------------------------------------------------------------- host side --
// One pool with its scales and the rows that go into it or come out of it.
static diopiError_t kvInt8Pool(const char* what, const char* name, const TensorView& x, const TensorView& pool, const TensorView& scale,
                               KvInt8Pool* o) {
  AMD_CHECK(x.defined() && pool.defined() && scale.defined(), "%s: %s: null tensor", what, name);
  AMD_CHECK(x.dtype == diopi_dtype_bfloat16 || x.dtype == diopi_dtype_float16 || x.dtype == diopi_dtype_float32, "%s: %s rows must be float16, bfloat16 or float32, got %s", what, name, dtypeName(x.dtype));
  AMD_CHECK(pool.dtype == diopi_dtype_int8, "%s: the %s pool must be int8, got %s", what, name, dtypeName(pool.dtype));
  AMD_CHECK(scale.dtype == diopi_dtype_float32, "%s: the %s scales must be float32, got %s", what, name, dtypeName(scale.dtype));
  AMD_CHECK(x.ndim == 3 && pool.ndim == 3 && scale.ndim == 2, "%s: %s rows and pool must be [n, kv_heads, head_dim], scales [slots, kv_heads]", what, name);
  AMD_CHECK(x.shape[1] == pool.shape[1] && x.shape[2] == pool.shape[2], "%s: %s rows are [%ld, %ld], those of the pool [%ld, %ld]", what, name,
            (long)x.shape[1], (long)x.shape[2], (long)pool.shape[1], (long)pool.shape[2]);
  AMD_CHECK(scale.shape[0] == pool.shape[0] && scale.shape[1] == pool.shape[1], "%s: %s scales must be [%ld, %ld]", what, name, (long)pool.shape[0], (long)pool.shape[1]);
  AMD_CHECK((x.stride[2] == 1 || x.shape[2] == 1) && (pool.stride[2] == 1 || pool.shape[2] == 1), "%s: %s head_dim must be contiguous", what, name);
  o->x = x.data, o->pool = pool.ptr<int8_t>(), o->scale = scale.ptr<float>();
  o->xToken = x.stride[0], o->xHead = x.stride[1];
  o->poolSlot = pool.stride[0], o->poolHead = pool.stride[1];
  o->scaleSlot = scale.stride[0], o->scaleHead = scale.stride[1];
  return diopiSuccess;
}

// Checks and arguments that both directions share. x: the rows, pool and scale: of K and V.
static diopiError_t kvInt8Args(const char* what, const TensorView (&x)[2], const TensorView (&pool)[2], const TensorView (&scale)[2], const TensorView& loc,
                               KvInt8Args* a) {
  AMD_TRY(kvInt8Pool(what, "k", x[0], pool[0], scale[0], &a->pool[0]));
  AMD_TRY(kvInt8Pool(what, "v", x[1], pool[1], scale[1], &a->pool[1]));
  AMD_CHECK(x[0].dtype == x[1].dtype, "%s: k rows are %s, v rows %s", what, dtypeName(x[0].dtype), dtypeName(x[1].dtype));
  for (int d = 0; d < 3; ++d)
    AMD_CHECK(x[0].shape[d] == x[1].shape[d] && pool[0].shape[d] == pool[1].shape[d], "%s: k and v shapes differ", what);
  AMD_CHECK(loc.defined() && loc.ndim == 1, "%s: the slots must be a tensor of one dim", what);
  AMD_CHECK(loc.dtype == diopi_dtype_int32 || loc.dtype == diopi_dtype_int64, "%s: the slots must be int32 or int64, got %s", what, dtypeName(loc.dtype));
  AMD_CHECK(loc.shape[0] == x[0].shape[0], "%s: %ld slots for %ld rows", what, (long)loc.shape[0], (long)x[0].shape[0]);
  AMD_CHECK(x[0].numel == 0 || pool[0].shape[0] > 0, "%s: the pool has no slots", what);
  AMD_CHECK(x[0].shape[0] < ((int64_t)1 << 31) && x[0].shape[1] <= (1 << 20) && x[0].shape[2] <= (1 << 20), "%s: extents exceed the launch limits", what);
  a->loc64 = loc.dtype == diopi_dtype_int64;
  a->tokens = x[0].shape[0], a->slots = pool[0].shape[0];
  AMD_CHECK(pool[0].shape[0] < ((int64_t)1 << 31), "%s: %ld slots exceed 2^31 - 1", what, (long)pool[0].shape[0]);
  a->heads = (int)x[0].shape[1], a->d = (int)x[0].shape[2];
  a->perHeads = 1.f / (float)a->heads;
  a->last = nullptr;
  return diopiSuccess;
}

// Whether all rows lie in whole 8-element pieces that can be loaded and stored at once.
static bool kvInt8Vector(const KvInt8Args& a, int64_t itemsize) {
  if (a.d % 8 != 0 || a.d > 256 || a.heads > (1 << 17)) return false;  // (heads: see kvTokenOf)
  int64_t bits16 = 0, bits8 = 0;
  for (const KvInt8Pool& o : a.pool) {
    // places within a workgroup's tokens, and heads within a slot, are products of 24-bit numbers below 2^31
    const int64_t token = o.xToken * kKvTokensPerWg, heads = std::max({o.xHead, o.poolHead, o.scaleHead});
    if (o.xToken >= (1 << 24) || heads >= (1 << 24) || token + heads * a.heads + a.d >= ((int64_t)1 << 31)) return false;
    bits16 |= (int64_t)reinterpret_cast<uintptr_t>(o.x) | o.xToken * itemsize | o.xHead * itemsize;
    bits8 |= (int64_t)reinterpret_cast<uintptr_t>(o.pool) | o.poolSlot | o.poolHead;
  }
  return (bits16 & 15) == 0 && (bits8 & 7) == 0;
}

// 32 or 64 rows to a workgroup: 64 where that leaves 256 workgroups (one per compute unit) for K and as many for V. us with 64, 128
// and 256: 8192 tokens of 32 heads written 45.3, 46.7, 45.4, read back 35.8, 36.6, 38.9; 15001 of 40 read back 83.8, 87.1, 91.8. 1777 tokens
// of 8 with 32 rows, from which the slots are looked up and looked through twice as often: 9.0, with 64 8.0.
static diopiError_t kvInt8Grid(const char* what, KvInt8Args* a, dim3* grid) {
  const int64_t rows = std::min<int64_t>(64, std::max<int64_t>(32, a->tokens * a->heads / 256));
  a->tokensPerWg = (int)std::min<int64_t>(kKvTokensPerWg, ceilDiv(rows, a->heads));
  const int64_t wgs = ceilDiv(a->tokens, a->tokensPerWg);
  AMD_CHECK(wgs < 1 << 24, "%s: %ld rows of %d heads exceed the launch limits", what, (long)a->tokens, a->heads);  // (2^32 threads)
  *grid = dim3((unsigned)wgs, 2);
  return diopiSuccess;
}

// NAME: kernels of one row width, of any, and their arguments behind the type and the width
#define KV_INT8_LAUNCH_TYPE(T, NAME, VEC, ...)                                                                                     \
  do {                                                                                                                             \
    if (!(VEC)) hipLaunchKernelGGL((NAME##AnyKernel<T __VA_OPT__(, ) __VA_ARGS__>), grid, dim3(kKvThreads), 0, stream, a);             \
    else if (a.d <= 64) hipLaunchKernelGGL((NAME##Kernel<T, 8 __VA_OPT__(, ) __VA_ARGS__>), grid, dim3(kKvThreads), 0, stream, a);     \
    else if (a.d <= 128) hipLaunchKernelGGL((NAME##Kernel<T, 16 __VA_OPT__(, ) __VA_ARGS__>), grid, dim3(kKvThreads), 0, stream, a);   \
    else hipLaunchKernelGGL((NAME##Kernel<T, 32 __VA_OPT__(, ) __VA_ARGS__>), grid, dim3(kKvThreads), 0, stream, a);                   \
  } while (0)
#define KV_INT8_LAUNCH(DTYPE, NAME, VEC, ...)                                                              \
  do {                                                                                                     \
    if (DTYPE == diopi_dtype_bfloat16) KV_INT8_LAUNCH_TYPE(bf16_t, NAME, VEC __VA_OPT__(, ) __VA_ARGS__);    \
    else if (DTYPE == diopi_dtype_float16) KV_INT8_LAUNCH_TYPE(half_t, NAME, VEC __VA_OPT__(, ) __VA_ARGS__); \
    else KV_INT8_LAUNCH_TYPE(float, NAME, VEC __VA_OPT__(, ) __VA_ARGS__);                                   \
  } while (0)

}  // namespace amd

using namespace amd;

extern "C" __attribute__((visibility("default"))) diopiError_t diopiDestIndexCopyKVPairInt8(
    diopiContextHandle_t ctx, diopiTensorHandle_t outKH, diopiTensorHandle_t outKScaleH, diopiConstTensorHandle_t kH,
    diopiTensorHandle_t outVH, diopiTensorHandle_t outVScaleH, diopiConstTensorHandle_t vH, diopiConstTensorHandle_t locH) {
  const char* what = "diopiDestIndexCopyKVPairInt8";
  hipStream_t stream;
  AMD_TRY(getStream(ctx, &stream));
  TensorView x[2], pool[2], scale[2], loc, dense;
  AMD_TRY(getView(outKH, &pool[0], "out_k"));
  AMD_TRY(getView(outKScaleH, &scale[0], "out_k_scale"));
  AMD_TRY(getView(kH, &x[0], "k"));
  AMD_TRY(getView(outVH, &pool[1], "out_v"));
  AMD_TRY(getView(outVScaleH, &scale[1], "out_v_scale"));
  AMD_TRY(getView(vH, &x[1], "v"));
  AMD_TRY(getView(locH, &loc, "dest_loc"));
  KvInt8Args a;
  AMD_TRY(kvInt8Args(what, x, pool, scale, loc, &a));
  if (x[0].numel == 0) return diopiSuccess;
  dim3 grid;
  AMD_TRY(kvInt8Grid(what, &a, &grid));
  AMD_TRY(makeContiguous(ctx, stream, loc, &dense));
  a.loc = dense.data;
  if (a.tokens > kKvScanTokens) {
    void* last = nullptr;
    AMD_TRY(requireWorkspace(ctx, a.slots * (int64_t)sizeof(int), &last));
    const dim3 perToken((unsigned)ceilDiv(a.tokens, kKvThreads));
    hipLaunchKernelGGL(kvInt8LastKernel<true>, perToken, dim3(kKvThreads), 0, stream, a, static_cast<int*>(last));
    hipLaunchKernelGGL(kvInt8LastKernel<false>, perToken, dim3(kKvThreads), 0, stream, a, static_cast<int*>(last));
    AMD_LAUNCH_CHECK();
    a.last = static_cast<const int*>(last);
  }
  const bool vector = kvInt8Vector(a, x[0].itemsize);
  if (a.last == nullptr) KV_INT8_LAUNCH(x[0].dtype, kvInt8Write, vector, true);
  else KV_INT8_LAUNCH(x[0].dtype, kvInt8Write, vector, false);
  AMD_LAUNCH_CHECK();
  return diopiSuccess;
}

extern "C" __attribute__((visibility("default"))) diopiError_t diopiIndexSelectKVPairInt8(
    diopiContextHandle_t ctx, diopiTensorHandle_t outKH, diopiTensorHandle_t outVH, diopiConstTensorHandle_t kH,
    diopiConstTensorHandle_t kScaleH, diopiConstTensorHandle_t vH, diopiConstTensorHandle_t vScaleH, diopiConstTensorHandle_t locH) {
  const char* what = "diopiIndexSelectKVPairInt8";
  hipStream_t stream;
  AMD_TRY(getStream(ctx, &stream));
  TensorView x[2], pool[2], scale[2], loc, dense;
  AMD_TRY(getView(outKH, &x[0], "out_k"));
  AMD_TRY(getView(outVH, &x[1], "out_v"));
  AMD_TRY(getView(kH, &pool[0], "k"));
  AMD_TRY(getView(kScaleH, &scale[0], "k_scale"));
  AMD_TRY(getView(vH, &pool[1], "v"));
  AMD_TRY(getView(vScaleH, &scale[1], "v_scale"));
  AMD_TRY(getView(locH, &loc, "index"));
  KvInt8Args a;
  AMD_TRY(kvInt8Args(what, x, pool, scale, loc, &a));
  if (x[0].numel == 0) return diopiSuccess;
  dim3 grid;
  AMD_TRY(kvInt8Grid(what, &a, &grid));
  AMD_TRY(makeContiguous(ctx, stream, loc, &dense));
  a.loc = dense.data;
  KV_INT8_LAUNCH(x[0].dtype, kvInt8Read, kvInt8Vector(a, x[0].itemsize));
  AMD_LAUNCH_CHECK();
  return diopiSuccess;
}
