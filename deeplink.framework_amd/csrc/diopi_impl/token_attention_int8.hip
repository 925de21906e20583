// Decode-step attention over an int8 KV pool for gfx950 (rows and scales: kv_int8.hip).
//
//   q [batch, heads, d] (fp16, bf16 or fp32), pool [slots, kv_heads, d] int8, scale [slots, kv_heads] fp32
//   out[b, h, :] = sum_t p_t (sv_t qv_t) / sum_t p_t,  p_t = exp(sk_t (q . qk_t) / sqrt(d) - max)
//
// The slot table, the lengths and what does not count (slots outside the pool) are those of token_attention.hip.
#include <algorithm>

#include "token_attention.hpp"

namespace amd {

struct TaInt8Args {
  TaArgs a;  // k and v: the int8 pools
  const float* kScale;
  const float* vScale;
  int64_t kScaleSlot, kScaleHead, vScaleSlot, vScaleHead;  // strides in elements
  int headsPerWg;  // K/V heads of a workgroup: 1, 2 or 4
  bool scaleVector;  // the scales of a workgroup's four heads can be read at once
  unsigned kStride, vStride;  // slot strides of the pools in bytes, as decodeInt8Kernel takes them
};

// ------------------------------------------------ head sizes of whole 16-byte pieces up to 256: the matrix pipe --
// Bound by memory: a row is d + 4 bytes, K and V alike. Both products of 32 tokens are matrix products (16x16x32, fp32 sums) with up
// to 16 query heads of a K/V head as columns; whole numbers up to 127 are exact in bf16 and in fp16, so the only things rounded
// are q (not at all: a 16-bit q is one operand and meets K in its own type, the 24 bits of fp32 are three of bf16) and the probabilities.
//   * S^T = K . Q^T: lane (token l % 16, group l / 16) needs 8 elements of its token's row for every product: it loads 16
//     adjacent bytes, which serve two of them (the order of the head's places along k is free as long as q has the same).
//   * a lane then holds eight tokens' scores of ONE head, so the softmax runs in the lane, and its probabilities are, as they lie,
//     the operand P^T of O^T += V^T . P^T. That operand wants eight tokens of V at one place of the head per lane: the lane loads
//     D / 16 adjacent bytes of each of its eight tokens, and the conversion to bf16 (one instruction per byte, whichever byte)
//     picks one byte out of each: V is turned round by the conversion that it needs anyway. So no row passes through LDS.
//   * the scale of K multiplies the score, that of V the probability, both in fp32; the product is cut into three parts of 8 bits,
//     each the rounding of what the ones before it leave: all 24 bits, for 16-bit results too (a sum that cancels shows what two
//     would lose; the third costs 1 %: 64 x (512 .. 4096), 32 heads, 230.7 -> 233.2 us). bf16 parts have the range of fp32, so
//     small weights keep theirs.
//   * the running maximum is followed at once (probabilities are at most one: a value near the type's largest does not
//     overflow); lanes exchange it only when one of them sees a larger one. Scores are rounded in units of log2 before it is taken
//     from them (K's scales in LDS hold 1 / (sqrt(d) ln 2) too): a multiply-add would leave the rounding of the maximum in the
//     exponent, which from 2^31 on is more than a number holds.
constexpr int kI8Waves = 4;
constexpr int kI8Tile = 32;   // tokens of a wave's step
constexpr int kI8Block = 512;  // tokens whose slots and scales a workgroup holds in LDS at once
constexpr int kI8Heads = 16;  // query heads a wave serves

template <typename T>
struct I8Parts {  // operands that hold q, and those that a probability is cut into
  static constexpr int kQ = std::is_same<T, float>::value ? 3 : 1;
  static constexpr int kP = 3;
};

// Bytes B0 of w0 and B1 of w1, signed, as two bf16 (exact: the upper half of the fp32 number).
template <int B0, int B1>
__device__ __forceinline__ uint32_t int8PairToBf16(uint32_t w0, uint32_t w1) {
  const float f0 = static_cast<float>(static_cast<int>(static_cast<int8_t>(w0 >> (8 * B0))));
  const float f1 = static_cast<float>(static_cast<int>(static_cast<int8_t>(w1 >> (8 * B1))));
  return __builtin_amdgcn_perm(__float_as_uint(f1), __float_as_uint(f0), 0x07060302u);
}

// The same as two operands of the product with q: fp16 q meets K in fp16 (exact too), anything else bf16.
template <typename T, int B0, int B1>
__device__ __forceinline__ uint32_t int8PairForQ(uint32_t w) {
  if constexpr (std::is_same<T, half_t>::value) {
    const float f0 = static_cast<float>(static_cast<int>(static_cast<int8_t>(w >> (8 * B0))));
    const float f1 = static_cast<float>(static_cast<int>(static_cast<int8_t>(w >> (8 * B1))));
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(f0, f1));
  } else {
    return int8PairToBf16<B0, B1>(w, w);
  }
}

template <int N>
struct I8Piece {  // N adjacent bytes of a row of V
  typedef uint32_t type __attribute__((ext_vector_type(N / 4)));
};

// The next part of each of eight numbers, and what it leaves of them.
__device__ __forceinline__ bf16x8 nextPart(float (&x)[8]) {
  bf16x8 part;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    part[i] = static_cast<bf16_t>(x[i]);
    x[i] -= static_cast<float>(part[i]);
  }
  return part;
}

// (The second launch bound: with three waves to a SIMD ten registers of D = 128 go to scratch, and 48 x (512 .. 4096), 8 K/V heads, takes 64 us, so 59.)
// D: head size the rows are laid out for; a.d is any multiple of 16 up to it: the pieces past the row's end repeat its first
// one, meet zeros of q, and give output places that are not stored. A workgroup's waves take x.headsPerWg K/V heads of the
// same tokens and share these out among the waves of a head.
template <typename T, int D>
__global__ __launch_bounds__(kI8Waves * 64, D == 256 ? 1 : 2) void decodeInt8Kernel(TaInt8Args x, T* __restrict__ out, float* __restrict__ partial) {
  const TaArgs& a = x.a;
  constexpr int PIECES = D / 64, RUN = D / 16, PQ = I8Parts<T>::kQ, PP = I8Parts<T>::kP;
  // V: a lane's RUN places of two tokens come in one load where they fit 16 bytes (see request)
  constexpr bool PAIRS = RUN < 16;
  typedef typename I8Piece<PAIRS ? 2 * RUN : RUN>::type VPiece;
  constexpr int VLOADS = PAIRS ? 4 : 8;
  extern __shared__ __attribute__((aligned(16))) float i8Lds[];
  __shared__ __attribute__((aligned(16))) int slots[kI8Block];  // of a block's tokens; negative: does not count
  __shared__ int badBuf[kI8Waves];
  __shared__ float stateBuf[kI8Waves][2][kI8Heads];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 15, quad = lane >> 4;

  // Workgroup ids go round the 8 XCDs. A unit is a (sequence, chunk); all its heads run next to each other on one XCD, whose L2
  // then fetches the line with a token's scales once for all of them. Units go sequence fastest, chunks from the last to the first,
  // each chunk's sequences one further on: the chunks of a long sequence then fall to different XCDs.
  const int f = blockIdx.x, idx = f >> 3;
  const int hw = x.headsPerWg, headGroups = (a.kvHeads + hw - 1) / hw * a.qGroups;
  const int hg = idx % headGroups, u = (idx / headGroups) * 8 + (f & 7);
  if (u >= a.batch * a.nsplit) return;  // the grid is rounded up to whole rounds of the XCDs
  const int level = u / a.batch, b = (u + level) % a.batch, split = a.nsplit - 1 - level;
  const int shares = kI8Waves / hw, share = wave / hw;
  const int firstHead = hg / a.qGroups * hw, kvh = min(firstHead + wave % hw, a.kvHeads - 1), g = hg % a.qGroups;
  const bool mine = firstHead + wave % hw < a.kvHeads;  // (the last group may be short of heads)
  // the block's scales: K of four heads, kI8Block floats each, then V; behind them the waves' sums for merging
  float* const scaleBuf = i8Lds;
  float* const i8Red = i8Lds + 2 * kI8Waves * kI8Block;
  const float* const scales = scaleBuf + wave % hw * kI8Block;
  const int perKv = a.heads / a.kvHeads, base = perKv / a.qGroups, rem = perKv % a.qGroups;
  const int h = kvh * perKv + g * base + min(g, rem), nq = base + (g < rem ? 1 : 0);  // the sharers are dealt evenly
  const int len = cutLength(a.bLen, b, a.len64, a.maxLen);
  const int begin = split * a.chunk;
  if (begin >= len && split != 0) return;  // split 0 still writes zeros for len == 0
  const int end = min(len, begin + a.chunk);
  const int64_t locBase = (int64_t)b * a.locRowStride + (a.maxLen - len);

  // q: product (p, s) of a row multiplies 8 places from placeOf(p) + 8 s on. All of it is asked for at once, and worked on when the
  // block's slots have been asked for too.
  auto placeOf = [&](int p) { return PIECES == 1 ? 16 * quad : 128 * (p >> 1) + 32 * quad + 16 * (p & 1); };
  constexpr int QLOADS = 8 / Vec16<T>::N;
  typename Vec16<T>::type qr[2 * PIECES][QLOADS];
#pragma unroll
  for (int p = 0; p < PIECES; ++p)
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const int e = placeOf(p) + 8 * s;
      const T* src = reinterpret_cast<const T*>(a.q) + b * a.qBatchStride + (h + min(col, nq - 1)) * a.qHeadStride + (e < a.d ? e : 0);
#pragma unroll
      for (int c = 0; c < QLOADS; ++c) qr[2 * p + s][c] = *(reinterpret_cast<const typename Vec16<T>::type*>(src) + c);
    }
  // Slots of the block's tokens: a thread looks up two (past the last: that token again) as two words, the second zero, or for 32-bit
  // indices the first again (a branch, or a conversion in one, would wait for the first load before it asks for the second). Without a
  // token: what q begins with, for nothing.
  int low[2], high[2];
  auto askSlots = [&](int block, int n) {
    const char* const locBytes = n > 0 ? static_cast<const char*>(a.bLoc) + ((locBase + block) << (a.loc64 ? 3 : 2)) : static_cast<const char*>(a.q);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const char* at = locBytes + ((int64_t)max(min((int)threadIdx.x + 256 * i, n - 1), 0) << (a.loc64 ? 3 : 2));
      low[i] = *reinterpret_cast<const int*>(at), high[i] = *reinterpret_cast<const int*>(at + (a.loc64 ? 4 : 0));
    }
    __builtin_amdgcn_sched_barrier(0);
  };
  askSlots(begin, min(kI8Block, end - begin));
  u32x4 qf[2 * PIECES][PQ];
#pragma unroll
  for (int p = 0; p < 2 * PIECES; ++p) {
    const bool have = col < nq && placeOf(p / 2) + 8 * (p % 2) < a.d;
    float v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = have ? static_cast<float>(qr[p][j / Vec16<T>::N][j % Vec16<T>::N]) : 0.f;
    if constexpr (std::is_same<T, half_t>::value) {
      f16x8 whole;
#pragma unroll
      for (int j = 0; j < 8; ++j) whole[j] = static_cast<half_t>(v[j]);
      qf[p][0] = __builtin_bit_cast(u32x4, whole);
    } else {
#pragma unroll
      for (int k = 0; k < PQ; ++k) qf[p][k] = __builtin_bit_cast(u32x4, nextPart(v));
    }
  }

  // Loads take whole 128-byte lines of 8 rows (or what of a row there is): K of two tiles of 8 tokens, in lanes 0 .. 7 and 8 .. 15
  // of each 16 the pieces 2 quad and 2 quad + 1, of which the lanes then swap one with the lane 8 aside; V of two tokens, one for each
  // eight lanes, of which the lanes keep one half and swap the other. (Rows read as the operands lie, 64 bytes of K and 8 of V to
  // a lane, twelve loads of a step instead of eight: 64 x (512 .. 4096) tokens, 32 heads, 359 us.)
  const int upperHalf = (lane >> 3) & 1;
  int kOff[PIECES];
#pragma unroll
  for (int p = 0; p < PIECES; ++p) {
    const int e = PIECES == 1 ? 16 * quad : 128 * (p >> 1) + 32 * quad + 16 * upperHalf;
    kOff[p] = e < a.d ? e : 0;
  }
  const int vAt = PAIRS ? (lane & 7) * 2 * RUN : col * RUN, vOff = vAt < a.d ? vAt : 0;
  const int8_t* const kBase = reinterpret_cast<const int8_t*>(a.k) + kvh * a.kHeadStride;
  const int8_t* const vBase = reinterpret_cast<const int8_t*>(a.v) + kvh * a.vHeadStride + vOff;
  struct Step {
    u32x4 k[2][PIECES];
    VPiece v[VLOADS];
  };
  auto request = [&](Step& s, int at) {
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int p = 0; p < PIECES; ++p) {
        const int token = at + 16 * t + (PIECES == 1 ? col : (lane & 7) + 8 * (p & 1));
        const int8_t* row = kBase + (uint64_t)((unsigned)slots[token] & 0x7fffffffu) * x.kStride;
        s.k[t][p] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(row + kOff[p]));
      }
#pragma unroll
    for (int i = 0; i < VLOADS; ++i) {
      const int token = at + (PAIRS ? 16 * (i >> 1) + 4 * quad + 2 * (i & 1) + upperHalf : 16 * (i >> 2) + 4 * quad + (i & 3));
      s.v[i] = __builtin_nontemporal_load(reinterpret_cast<const VPiece*>(vBase + (uint64_t)((unsigned)slots[token] & 0x7fffffffu) * x.vStride));
    }
    __builtin_amdgcn_sched_barrier(0);  // nothing of the step before is touched (and waited for) ahead of these loads
  };
  // `own` in the lanes of `BANKS` (0xc: 8 .. 15 of each 16, 0x3: 0 .. 7) replaced by what the lane 8 aside has in `other`
  auto swapped = [](uint32_t own, uint32_t other, auto banks) {
    return (uint32_t)__builtin_amdgcn_update_dpp((int)own, (int)other, 0x128 /* rotate 16 lanes by 8 */, 0xf, decltype(banks)::value, false);
  };
  constexpr std::integral_constant<int, 0xc> kUpper{};
  constexpr std::integral_constant<int, 0x3> kLower{};

  f32x4 acc[RUN];
#pragma unroll
  for (int t = 0; t < RUN; ++t) acc[t] = f32x4{0.f, 0.f, 0.f, 0.f};
  // this lane's head: the largest score (in units of log2), and what scores are taken against (that, or 0 while there is none)
  float m = -INFINITY, mRef = 0.f, l = 0.f;
  auto multiply = [&](Step& s, int at, bool all) {  // all: every one of the tokens counts
    f32x4 ks[2], vs[2], s4[2];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      ks[t] = *reinterpret_cast<const f32x4*>(scales + at + 16 * t + 4 * quad);
      vs[t] = *reinterpret_cast<const f32x4*>(scales + kI8Waves * kI8Block + at + 16 * t + 4 * quad);
      s4[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int p = 0; p < PIECES; ++p)
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          auto word = [&](int c) {  // of the lane's token: even p, its piece 2 quad of a line, odd p, the next
            if (PIECES == 1) return s.k[t][0][c];
            return p & 1 ? swapped(s.k[t][p][c], s.k[t][p - 1][c], kLower) : swapped(s.k[t][p][c], s.k[t][p + 1 < PIECES ? p + 1 : p][c], kUpper);
          };
          const uint32_t w0 = word(2 * half), w1 = word(2 * half + 1);
          const u32x4 kf = {int8PairForQ<T, 0, 1>(w0), int8PairForQ<T, 2, 3>(w0), int8PairForQ<T, 0, 1>(w1), int8PairForQ<T, 2, 3>(w1)};
          if constexpr (std::is_same<T, half_t>::value) {
            s4[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, kf), __builtin_bit_cast(f16x8, qf[2 * p + half][0]), s4[t], 0, 0, 0);
          } else {
#pragma unroll
            for (int k = 0; k < PQ; ++k)
              s4[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, kf), __builtin_bit_cast(bf16x8, qf[2 * p + half][k]), s4[t], 0, 0, 0);
          }
        }
    }
    float sc[8], w[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      sc[i] = s4[i >> 2][i & 3] * ks[i >> 2][i & 3];
      w[i] = vs[i >> 2][i & 3];
    }
    if (!all) {
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const int4 m4 = *reinterpret_cast<const int4*>(slots + at + 16 * t + 4 * quad);
        const int mine[4] = {m4.x, m4.y, m4.z, m4.w};
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (mine[i] < 0) sc[4 * t + i] = -INFINITY, w[4 * t + i] = 0.f;  // (slot 0, which stands in, may hold any scale)
      }
    }
    float mt = sc[0];
#pragma unroll
    for (int i = 1; i < 8; ++i) mt = fmaxf(mt, sc[i]);
    if (__builtin_amdgcn_ballot_w64(mt > m) != 0) {
      auto sw = __builtin_amdgcn_permlane32_swap(__float_as_uint(mt), __float_as_uint(mt), false, false);
      mt = fmaxf(__uint_as_float(sw[0]), __uint_as_float(sw[1]));
      sw = __builtin_amdgcn_permlane16_swap(__float_as_uint(mt), __float_as_uint(mt), false, false);
      mt = fmaxf(__uint_as_float(sw[0]), __uint_as_float(sw[1]));
      if (mt > m) {
        const float corr = m == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m - mt);  // (no maximum yet: the sums are 0, or NaN)
        m = mRef = mt;
        l *= corr;
#pragma unroll
        for (int t = 0; t < RUN; ++t)
#pragma unroll
          for (int i = 0; i < 4; ++i) acc[t][i] *= corr;
      }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float e = __builtin_amdgcn_exp2f(behindRounded(sc[i], mRef));
      l += e;
      w[i] *= e;
    }
    bf16x8 pf[PP];
#pragma unroll
    for (int k = 0; k < PP; ++k) pf[k] = nextPart(w);
    // V of the lane's eight tokens at its RUN places, RUN / 4 words each
    uint32_t v[8][RUN / 4];
#pragma unroll
    for (int i = 0; i < VLOADS; ++i)
#pragma unroll
      for (int c = 0; c < RUN / 4; ++c) {
        if constexpr (PAIRS) {
          v[2 * i][c] = swapped(s.v[i][c], s.v[i][RUN / 4 + c], kUpper);
          v[2 * i + 1][c] = swapped(s.v[i][RUN / 4 + c], s.v[i][c], kLower);
        } else {
          v[i][c] = s.v[i][c];
        }
      }
    staticFor<RUN>([&](auto t) {
      constexpr int W = t.value / 4, B = t.value % 4;
      u32x4 o;
#pragma unroll
      for (int j = 0; j < 4; ++j) o[j] = int8PairToBf16<B, B>(v[2 * j][W], v[2 * j + 1][W]);
#pragma unroll
      for (int k = 0; k < PP; ++k) acc[t.value] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, o), pf[k], acc[t.value], 0, 0, 0);
    });
  };

  for (int block = begin; block < end; block += kI8Block) {
    const int n = min(kI8Block, end - block);
    if (block != begin) __syncthreads();  // every wave is done with the block before
    if (block != begin) askSlots(block, n);
    unsigned slot[2];
    bool bad = false;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      // slots outside the pool are skipped, never dereferenced
      const bool in = low[i] >= 0 && low[i] < (int)a.slots && (!a.loc64 || high[i] == 0);
      const bool counts = in && (int)threadIdx.x + 256 * i < n;
      slot[i] = in ? (unsigned)low[i] : 0u;
      slots[threadIdx.x + 256 * i] = counts ? (int)slot[i] : (int)(slot[i] | 0x80000000u);
      bad |= !in;
    }
    const bool waveBad = __builtin_amdgcn_ballot_w64(bad) != 0;
    if (lane == 0) badBuf[wave] = waveBad;
    __syncthreads();
    const bool clean = !(badBuf[0] | badBuf[1] | badBuf[2] | badBuf[3]);
    // scales of the workgroup's heads, before the rows: loads return to a wave in issue order
    float ksv[2][kI8Waves], vsv[2][kI8Waves];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const float* kAt = x.kScale + (uint64_t)slot[i] * (unsigned)x.kScaleSlot;
      const float* vAt = x.vScale + (uint64_t)slot[i] * (unsigned)x.vScaleSlot;
      if (x.scaleVector) {
        const f32x4 k4 = *reinterpret_cast<const f32x4*>(kAt + firstHead), v4 = *reinterpret_cast<const f32x4*>(vAt + firstHead);
#pragma unroll
        for (int w = 0; w < kI8Waves; ++w) ksv[i][w] = k4[w], vsv[i][w] = v4[w];
      } else {
#pragma unroll
        for (int w = 0; w < kI8Waves; ++w) {  // (of four heads also where there are fewer: loads that nothing waits for here, the loop below would)
          const int head = min(firstHead + w, a.kvHeads - 1);
          ksv[i][w] = kAt[head * x.kScaleHead], vsv[i][w] = vAt[head * x.vScaleHead];
        }
      }
    }
    const int perShare = ((n + shares - 1) / shares + kI8Tile - 1) / kI8Tile * kI8Tile;  // whole steps
    const int from = share * perShare, to = mine ? min(n, from + perShare) : from;
    Step s0, s1;
    request(s0, from);  // (also where the wave has no step: all of the block's slots can be read, and a branch would cost as below)
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int w = 0; w < kI8Waves; ++w) {
        scaleBuf[w * kI8Block + threadIdx.x + 256 * i] = ksv[i][w] * a.scaleLog2e;
        scaleBuf[(kI8Waves + w) * kI8Block + threadIdx.x + 256 * i] = vsv[i][w];
      }
    __syncthreads();
    // (the last one or two steps stand by themselves: a branch around the loads of the loop would make every wait one for all of them)
    int at = from;
    for (; at + 2 * kI8Tile < to; at += 2 * kI8Tile) {
      request(s1, at + kI8Tile);
      multiply(s0, at, clean);
      request(s0, at + 2 * kI8Tile);
      multiply(s1, at + kI8Tile, clean);
    }
    if (at + kI8Tile < to) {
      request(s1, at + kI8Tile);
      multiply(s0, at, clean);
      multiply(s1, at + kI8Tile, clean && at + 2 * kI8Tile <= n);
    } else if (at < to) {
      multiply(s0, at, clean && at + kI8Tile <= n);
    }
  }

  // every lane group holds its own share of l; O^T lies in the lanes as (head = column, places runOf(4 quad + i) + t)
  {
    auto sw = __builtin_amdgcn_permlane32_swap(__float_as_uint(l), __float_as_uint(l), false, false);
    l = __uint_as_float(sw[0]) + __uint_as_float(sw[1]);
    sw = __builtin_amdgcn_permlane16_swap(__float_as_uint(l), __float_as_uint(l), false, false);
    l = __uint_as_float(sw[0]) + __uint_as_float(sw[1]);
  }
  auto runOf = [](int c) { return PAIRS ? (c & 7) * 2 * RUN + (c >> 3) * RUN : c * RUN; };  // the first of lane c's places of V
  if (l != l && m == -INFINITY) m = 0.f;  // scores that are not numbers alone: as a maximum of minus infinity they would be left out
  auto store = [&](int j, int e, float mAll, float lAll, f32x4 o) {  // four places of head h + j
    if (a.nsplit == 1) {
      const float inv = lAll == 0.f ? 0.f : 1.f / lAll;
      typedef T Quad __attribute__((ext_vector_type(4)));
      Quad r;
#pragma unroll
      for (int c = 0; c < 4; ++c) r[c] = static_cast<T>(o[c] * inv);
      storeElements(out + ((int64_t)b * a.heads + h + j) * a.d + e, r);
    } else {
      float* dst = partial + (((int64_t)b * a.heads + h + j) * a.nsplit + split) * (2 + a.d);
      if (e == 0) dst[0] = mAll, dst[1] = lAll;
#pragma unroll
      for (int c = 0; c < 4; ++c) dst[2 + e + c] = o[c];
    }
  };
  if (shares == 1) {
    if (mine && col < nq) {
      staticFor<RUN / 4>([&](auto r) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int e = runOf(4 * quad + i) + 4 * r.value;
          if (e < a.d) store(col, e, m, l, f32x4{acc[4 * r.value][i], acc[4 * r.value + 1][i], acc[4 * r.value + 2][i], acc[4 * r.value + 3][i]});
        }
      });
    }
    return;
  }
  constexpr int kRedRow = D + 4;  // floats per head
  if (mine && col < nq) {
    if (quad == 0) stateBuf[wave][0][col] = m, stateBuf[wave][1][col] = l;
    staticFor<RUN / 4>([&](auto r) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        *reinterpret_cast<f32x4*>(i8Red + (wave * nq + col) * kRedRow + runOf(4 * quad + i) + 4 * r.value) =
            f32x4{acc[4 * r.value][i], acc[4 * r.value + 1][i], acc[4 * r.value + 2][i], acc[4 * r.value + 3][i]};
    });
  }
  __syncthreads();
  if (!mine) return;
  for (int i = share * 64 + lane; i < nq * (D / 4); i += shares * 64) {
    const int j = i / (D / 4), e = (i % (D / 4)) * 4;
    if (e >= a.d) continue;
    float mAll = -INFINITY, lAll = 0.f;
    for (int k = wave % hw; k < kI8Waves; k += hw) mAll = fmaxf(mAll, stateBuf[k][0][j]);
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
    for (int k = wave % hw; k < kI8Waves; k += hw) {
      const float mk = stateBuf[k][0][j];
      const float wk = mk == -INFINITY ? 0.f : exp2f(mk - mAll);
      lAll += stateBuf[k][1][j] * wk;
      const f32x4 v = *reinterpret_cast<const f32x4*>(i8Red + (k * nq + j) * kRedRow + e);
#pragma unroll
      for (int c = 0; c < 4; ++c) o[c] += v[c] * wk;
    }
    store(j, e, mAll, lAll, o);
  }
}

// ---------------------------------------------------------------- host side --
static diopiError_t int8Pool(const char* name, const TensorView& q, const TensorView& pool, const TensorView& scale) {
  AMD_CHECK(pool.defined() && pool.ndim == 3 && scale.defined() && scale.ndim == 2,
            "int8 token attention: %s must be [slots, kv_heads, head_dim] with scales [slots, kv_heads]", name);
  AMD_CHECK(pool.dtype == diopi_dtype_int8, "int8 token attention: %s must be int8, got %s", name, dtypeName(pool.dtype));
  AMD_CHECK(scale.dtype == diopi_dtype_float32, "int8 token attention: the scales of %s must be float32, got %s", name, dtypeName(scale.dtype));
  AMD_CHECK(pool.shape[0] > 0, "int8 token attention: the %s pool has no slots", name);
  AMD_CHECK(scale.shape[0] == pool.shape[0] && scale.shape[1] == pool.shape[1], "int8 token attention: the scales of %s must be [%ld, %ld]", name,
            (long)pool.shape[0], (long)pool.shape[1]);
  AMD_CHECK(pool.shape[1] > 0 && q.shape[1] % pool.shape[1] == 0, "int8 token attention: %ld heads are not a multiple of %ld kv heads",
            (long)q.shape[1], (long)pool.shape[1]);
  AMD_CHECK(pool.shape[2] == q.shape[2], "int8 token attention: head_dim mismatch (%ld vs %ld)", (long)pool.shape[2], (long)q.shape[2]);
  AMD_CHECK(pool.stride[2] == 1 || pool.shape[2] == 1, "int8 token attention: the head_dim of %s must be contiguous", name);
  return diopiSuccess;
}

// Heads of a workgroup and tokens of a chunk. steps: of 32 tokens of a head, of all sequences at the longest one's length; a wave
// gets one of them where there are few (its step takes 0.5 us, whoever waits for rows does nothing else), and up to 16 where
// there are many (what a workgroup does before its first step, and its partial results, are then spread over more). With four
// heads to a workgroup a wave reads 512 adjacent bytes of a token with the other three, and one lane the scales of all four: 64 x
// (512 .. 4096) tokens, 32 heads of 128, 234 us, with one head 365 (48, 8 heads 59 and 82). Few steps are better dealt over the
// waves of a head: 1 x 1777 tokens, 8 heads, one step to a wave, 10.0 with one head, 11.1 with four.
// us at 1, 2, 4, 8, 16 steps to a wave: 1 x 4096, 8 heads 10.3, 11.1, 13.4, 17.5, 24.8; 1 x 8192 13.9, 12.9, 15.0, 17.9, 25.4; 1 x 16384
// 23.9, 19.7, 18.3, 19.5, 25.6; 8 x 4096 34, 27, 22.7, 20.8, 26.0; 16 x (1000 .. 8000) 76, 55, 47, 47, 47; 48 x (512 .. 4096) 109, 75, 66, 59, 68;
// 32 heads, 64 x (512 .. 4096) 550, 357, 283, 247, 232. Heads of 256: a SIMD holds one wave instead of two, and a step takes twice as
// long: 16 x (512 .. 4096), 8 heads 92, 65, 58, 55, 46. Next to the line between 8 and 16 (steps for a compute unit in brackets), 8 heads of
// 128, two sets of lengths of 512 .. 4096: 40 sequences [160] 54 and 49, 52 and 49; 48 [192] 59 and 67, 60 and 58; 52 [208] 62 and 67, 68 and 69;
// 56 [224] 67 and 74, 70 and 75; 64 [256] 78 and 77, 80 and 79; 96 [384] 118 and 113, 114 and 106; all of 4096: 48 88 and 81, 56 102 and 99, 64 116 and
// 105. 32 heads, 14 [224] 64 and 71, 16 [256] 69 and 74, 32 [512] 130 and 133, 64 [1024] 247 and 232; of 64, 32 [512] 101 and 108. Which one a set of
// lengths likes turns on how its last round of workgroups comes out; from 256 on even lengths and the large batches are better in 16.
static void chooseShares(TaInt8Args* x, int64_t len, int D) {
  TaArgs& a = x->a;
  const int64_t steps = (int64_t)a.kvHeads * a.qGroups * a.batch * ceilDiv(len, kI8Tile) * (D == 256 ? 4 : 1);
  const int64_t perUnit = steps / computeUnits();
  const int perWave = perUnit < 6 ? 1 : perUnit < 12 ? 2 : perUnit < 24 ? 4 : perUnit < 224 ? 8 : 16;
  // (heads in twos and fours leave waves without a head: of 5 in fours 3, 74 us where twos take 68)
  const int fits = a.kvHeads % 4 == 0 || a.kvHeads == 3 || a.kvHeads > 8 ? 4 : a.kvHeads >= 2 ? 2 : 1;
  x->headsPerWg = std::min(fits, perWave);
  int64_t tokens = (int64_t)perWave * kI8Tile * kI8Waves / x->headsPerWg;
  // short sequences in one chunk, without the launch that merges: 16 x (1 .. 300), 8 heads of 64, 9.4 -> 7.6; 64 x (100 .. 500), 32 heads
  // 41.1 -> 38.6
  if (len <= kI8Block && perWave >= 8) {
    tokens = len;
  } else if (len <= 384 && a.batch >= 8) {
    x->headsPerWg = 1, tokens = len;
  }
  const int64_t step = kI8Tile * kI8Waves / x->headsPerWg;
  tokens = std::max<int64_t>(std::min<int64_t>(tokens, kI8Block), ceilDiv(len, kTaMaxSplit));
  a.chunk = (int)(ceilDiv(tokens, step) * step);
  a.nsplit = (int)ceilDiv(len, a.chunk);
}

static diopiError_t decodeInt8(diopiContextHandle_t ctx, hipStream_t stream, TaInt8Args x, const TensorView& q, void* out) {
  TaArgs& a = x.a;
  const int64_t perKv = a.heads / a.kvHeads, len = std::max(a.maxLen, 1);
  a.qGroups = (int)ceilDiv(perKv, kI8Heads);
  if (!q.aligned16() || ((q.stride[0] | q.stride[1]) * q.itemsize) % 16 != 0) {  // the kernel reads whole 16 bytes: a dense copy of q
    diopiTensorHandle_t th = nullptr;
    TensorView dense;
    AMD_TRY(requireTensor(ctx, q.shape, q.ndim, q.dtype, &th, &dense));
    AMD_TRY(stridedCopy(stream, q, dense));
    a.q = dense.data, a.qBatchStride = dense.stride[0], a.qHeadStride = dense.stride[1];
  }
  const int D = a.d <= 64 ? 64 : a.d <= 128 ? 128 : 256;
  chooseShares(&x, len, D);
  x.scaleVector = x.headsPerWg == 4 && a.kvHeads % 4 == 0 && x.kScaleHead == 1 && x.vScaleHead == 1 && (x.kScaleSlot | x.vScaleSlot) % 4 == 0 &&
                  ((reinterpret_cast<uintptr_t>(x.kScale) | reinterpret_cast<uintptr_t>(x.vScale)) & 15) == 0;
  x.kStride = (unsigned)a.kSlotStride, x.vStride = (unsigned)a.vSlotStride;
  const int64_t headGroups = ceilDiv(a.kvHeads, x.headsPerWg) * a.qGroups;
  float* partial = nullptr;
  if (a.nsplit > 1) {
    void* ws = nullptr;
    AMD_TRY(requireWorkspace(ctx, (int64_t)a.batch * a.heads * a.nsplit * (2 + a.d) * (int64_t)sizeof(float), &ws));
    partial = static_cast<float*>(ws);
  }
  const int64_t wgs = ceilDiv((int64_t)a.batch * a.nsplit, 8) * 8 * headGroups;
  AMD_CHECK(wgs < 1 << 24, "int8 token attention: %ld workgroups exceed the grid limits", (long)wgs);  // (2^32 threads)
  const int lds = 2 * kI8Waves * kI8Block * (int)sizeof(float) + (x.headsPerWg == kI8Waves ? 0 : kI8Waves * (int)std::min<int64_t>(perKv, kI8Heads) * (D + 4) * (int)sizeof(float));
#define INT8_CALL(T, SIZE)                                                                                              \
  do {                                                                                                                  \
    AMD_HIP(allowDynamicLds(reinterpret_cast<const void*>(decodeInt8Kernel<T, SIZE>), lds));                             \
    hipLaunchKernelGGL((decodeInt8Kernel<T, SIZE>), dim3((unsigned)wgs), dim3(kI8Waves * 64), lds, stream, x, static_cast<T*>(out), partial); \
  } while (0)
#define INT8_SIZES(T) \
  if (D == 64) INT8_CALL(T, 64); else if (D == 128) INT8_CALL(T, 128); else INT8_CALL(T, 256)
  if (q.dtype == diopi_dtype_bfloat16) { INT8_SIZES(bf16_t); }
  else if (q.dtype == diopi_dtype_float16) { INT8_SIZES(half_t); }
  else { INT8_SIZES(float); }
#undef INT8_SIZES
#undef INT8_CALL
  AMD_LAUNCH_CHECK();
  return a.nsplit > 1 ? mergeChunks(stream, q.dtype, out, partial, a, a.batch) : diopiSuccess;
}

}  // namespace amd

using namespace amd;

extern "C" __attribute__((visibility("default"))) diopiError_t diopiTokenDecodeAttentionInt8Inference(
    diopiContextHandle_t ctx, diopiTensorHandle_t outH, diopiConstTensorHandle_t qH, diopiConstTensorHandle_t kH,
    diopiConstTensorHandle_t kScaleH, diopiConstTensorHandle_t vH, diopiConstTensorHandle_t vScaleH, diopiConstTensorHandle_t locH,
    diopiConstTensorHandle_t startH, diopiConstTensorHandle_t lenH, int maxInputLen) {
  hipStream_t stream;
  AMD_TRY(getStream(ctx, &stream));
  TaViews t;
  TensorView out, kScale, vScale;
  AMD_TRY(getView(outH, &out, "out"));
  AMD_TRY(getView(qH, &t.q, "q"));
  AMD_TRY(getView(kH, &t.k, "k"));
  AMD_TRY(getView(kScaleH, &kScale, "k_scale"));
  AMD_TRY(getView(vH, &t.v, "v"));
  AMD_TRY(getView(vScaleH, &vScale, "v_scale"));
  AMD_TRY(getView(locH, &t.loc, "b_loc"));
  AMD_TRY(getView(startH, &t.start, "b_start_loc"));
  AMD_TRY(getView(lenH, &t.len, "b_seq_len"));
  TaInt8Args x;
  TaArgs& a = x.a;
  AMD_TRY(tableArgs(t, maxInputLen, &a));
  AMD_TRY(int8Pool("k", t.q, t.k, kScale));
  AMD_TRY(int8Pool("v", t.q, t.v, vScale));
  for (int d = 0; d < 3; ++d) AMD_CHECK(t.v.shape[d] == t.k.shape[d], "int8 token attention: k and v shapes differ");
  AMD_CHECK(out.defined() && out.dtype == t.q.dtype && out.ndim == 3 && out.isContiguous(), "int8 token attention: out must be a dense tensor shaped like q");
  for (int d = 0; d < 3; ++d) AMD_CHECK(out.shape[d] == t.q.shape[d], "int8 token attention: out must be shaped like q");
  AMD_CHECK(t.q.shape[2] <= kTaGenericMaxD, "int8 token attention: head_dim %ld exceeds %d", (long)t.q.shape[2], kTaGenericMaxD);
  a.k = t.k.data, a.v = t.v.data;
  a.kSlotStride = t.k.stride[0], a.kHeadStride = t.k.stride[1], a.vSlotStride = t.v.stride[0], a.vHeadStride = t.v.stride[1];
  a.slots = t.k.shape[0], a.kvHeads = (int)t.k.shape[1];
  x.kScale = kScale.ptr<float>(), x.vScale = vScale.ptr<float>();
  x.kScaleSlot = kScale.stride[0], x.kScaleHead = kScale.stride[1], x.vScaleSlot = vScale.stride[0], x.vScaleHead = vScale.stride[1];
  if (t.q.numel == 0) return diopiSuccess;
  AMD_CHECK(a.batch <= 65535, "int8 token attention: batch %d exceeds the grid limits", a.batch);
  // rows of whole 16-byte pieces, slot numbers in 31 bits: the matrix pipe
  const int64_t bits = (int64_t)reinterpret_cast<uintptr_t>(a.k) | (int64_t)reinterpret_cast<uintptr_t>(a.v) | a.kSlotStride | a.kHeadStride | a.vSlotStride |
                       a.vHeadStride | a.d;
  const int64_t widest = std::max({a.kSlotStride, a.vSlotStride, x.kScaleSlot, x.vScaleSlot});
  if ((bits & 15) == 0 && a.d <= 256 && a.slots <= 0x7fffffff && widest <= 0xffffffffll) return decodeInt8(ctx, stream, x, t.q, out.data);
  TaAnyArgs any{};
  any.a = a, any.kScale = x.kScale, any.vScale = x.vScale;
  any.kScaleSlot = x.kScaleSlot, any.kScaleHead = x.kScaleHead, any.vScaleSlot = x.vScaleSlot, any.vScaleHead = x.vScaleHead;
  TaPartials own;
  AMD_TRY(walkAny(ctx, stream, any, t.q.dtype, out.data, true, &own));
  return own.nsplit == 0 ? diopiSuccess : mergeShares(stream, a, t.q.dtype, out.data, nullptr, 0, own, 0);
}
