// Decode-step attention of a batch whose sequences all begin with the same tokens (a system prompt, a document), kept once in
// the paged pool, for gfx950.
//
//   q [batch, heads, d], k, v [slots, kv_heads, d]      as in token_attention.hip
//   prefix_loc [n]                                       the slots of the shared tokens
//   b_loc, b_seq_len                                     each sequence's own tokens behind them
//
// out[b, h, :] = softmax over the n shared tokens and the b_seq_len[b] own ones of q . k / sqrt(d), times v.
#include <algorithm>

#include "token_attention.hpp"

namespace amd {

struct TaPrefixArgs {
  TaArgs a;
  const void* loc;  // slots of the shared tokens
  bool loc64;
  int len;
  int chunk, nsplit;          // of the shared tokens
  int groups;                 // of columns
  unsigned kStride, vStride;  // slot strides of the pools in bytes
};

// ------------------------------------------------ head rows of whole 16-byte pieces up to 256 elements: the matrix pipe --
// The shared tokens see the same K and V from every sequence, so a K/V head's columns are the query heads that share it of ALL
// sequences: S^T = K . Q^T and O^T += V^T . P^T with many columns for one read of a row. Partial results (maximum, sum, weighted
// sum of V) of each chunk of the prefix go to workspace; those of the sequences' own tokens come from the kernels of
// diopiTokenDecodeAttentionInference, which end on the shared tokens' where the own ones are one chunk; a last launch merges the partial
// results of both where they are more. (fp32 rows of more than 512 bytes, which those do not take: token_attention_any.hip.)
//
// Long prefixes are bound by memory, every shared row read once (for each group of columns), and, with many columns, by the matrix
// pipe and the exponentials; short ones by the launches and the latency of slots, then rows.
//
// ------------------------------------------------ fp32 --
// Rows go from the pool into the registers that the products (16x16x4) read, whole 128-byte lines of 8 rows in a load: K as in
// token_attention_int8.hip (two lanes swap a piece of 16 bytes), of V a lane takes 16 adjacent bytes of each of its four tokens.
//   * the running maximum is followed at once, so a probability is at most one.
//   * the first walk multiplies V as it is: infinities and NaN in it, or in slot 0 for a slot outside the pool, against
//     probabilities that are zero leave sums that are not finite, and the wave then walks again with care: rows that do not count
//     are zeros, what is not finite meets a one for each probability that is not zero. So it does where the maximum is far from
//     zero (kPxFar): the first walk's exponents are multiply-adds, which keep what the maximum lost in rounding.
// Four waves share a chunk's tokens and meet in LDS, a lane always adding to what is its own. 16 000 tokens, 32 heads of 128, 24
// sequences: 132 us, 4.0 TB/s; two tiles of columns share a read with heads of 64 (with 128 that takes more registers than there are).
constexpr int kPxWaves = 4;
constexpr int kPxBlock = 2048;    // tokens whose slots a workgroup holds in LDS at once
constexpr int kPxMaxSplit = 256;  // chunks of the prefix
// Maxima up to this size (in units of log2) are off by at most 1/8, so are then the exponents of a walk without care, which does
// not matter: all of a sum's are, and fp16 probabilities, at most 2^15, have room for it. From 2^31 on nothing would be left of them.
constexpr float kPxFar = 0x1p22f;
__device__ __forceinline__ bool pxFar(float m) { return fabsf(m) > kPxFar && m != -INFINITY; }

template <int D>
struct PxShape {
  static constexpr int KP = D / 16;   // 16-byte pieces of K per lane
  static constexpr int RUN = D / 16;  // places of V per lane
  static constexpr int VP = D / 64;   // 16-byte pieces of V per lane and token
  // place t of lane c's places of V in the head
  static __device__ __forceinline__ int place(int c, int t) { return t / 4 * 64 + c * 4 + t % 4; }
};

// D: head size the rows are laid out for; a.d is any whole number of 16-byte pieces up to it. NC: column tiles of 16.
template <int D, int NC>
__global__ __launch_bounds__(kPxWaves * 64, 1) void decodePrefixFloatKernel(TaPrefixArgs x, float* __restrict__ partial) {
  using S = PxShape<D>;
  constexpr int TOKENS = 16, KP = S::KP, RUN = S::RUN, VP = S::VP;  // TOKENS: of a wave's step
  const TaArgs& a = x.a;
  extern __shared__ __attribute__((aligned(16))) f32x4 pxLds[];  // sums on their way to the waves that add them up
  __shared__ __attribute__((aligned(16))) int slots[kPxBlock];  // of a block's tokens; negative: does not count
  __shared__ int badBuf[kPxWaves];
  __shared__ float stateBuf[kPxWaves][NC][2][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 15, quad = lane >> 4, upperHalf = (lane >> 3) & 1;

  // Workgroup ids go round the 8 XCDs. A unit is a (chunk, K/V head); its groups of columns read the same rows and run next to
  // each other on one XCD.
  const int f = blockIdx.x, idx = f >> 3;
  const int perKv = a.heads / a.kvHeads, columns = a.batch * perKv, tiles = (columns + 15) / 16, groups = x.groups;
  const int group = idx % groups, u = (idx / groups) * 8 + (f & 7);
  if (u >= a.kvHeads * x.nsplit) return;  // the grid is rounded up to whole rounds of the XCDs
  const int kvh = u % a.kvHeads, split = u / a.kvHeads;
  const int begin = split * x.chunk, end = min(x.len, begin + x.chunk);

  // tiles of columns are dealt out evenly to the groups: up to NC to one
  const int firstTile = (int)((int64_t)group * tiles / groups), lastTile = (int)((int64_t)(group + 1) * tiles / groups);

  // q of the columns: column c of the K/V head is its query head c % perKv in sequence c / perKv. Piece p holds four places from
  // the byte 128 (p / 2) + 32 quad + 16 (p % 2) of the row on.
  f32x4 qf[NC][KP];
  int pairOf[NC];  // row of the partial results of this lane's column, or -1
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    const int column = (firstTile + c) * 16 + col;
    const bool have = firstTile + c < lastTile && column < columns;
    const int b = have ? column / perKv : 0, h = kvh * perKv + (have ? column % perKv : 0);
    pairOf[c] = have ? b * a.heads + h : -1;
    const float* src = reinterpret_cast<const float*>(a.q) + b * a.qBatchStride + h * a.qHeadStride;
#pragma unroll
    for (int p = 0; p < KP; ++p) {
      const int e = 32 * (p >> 1) + 8 * quad + 4 * (p & 1);
      qf[c][p] = *reinterpret_cast<const f32x4*>(src + (e < a.d ? e : 0));
      if (!have || e >= a.d) qf[c][p] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
  }

  int kOff[KP], vOff[VP];  // bytes; pieces past the row's end repeat its first one
  const int rowBytes = a.d * (int)sizeof(float);
#pragma unroll
  for (int p = 0; p < KP; ++p) {
    const int e = 128 * (p >> 1) + 32 * quad + 16 * upperHalf;
    kOff[p] = e < rowBytes ? e : 0;
  }
#pragma unroll
  for (int p = 0; p < VP; ++p) {
    const int e = 256 * p + 16 * col;
    vOff[p] = e < rowBytes ? e : 0;
  }
  const char* const kBase = reinterpret_cast<const char*>(reinterpret_cast<const float*>(a.k) + kvh * a.kHeadStride);
  const char* const vBase = reinterpret_cast<const char*>(reinterpret_cast<const float*>(a.v) + kvh * a.vHeadStride);

  struct Step {
    u32x4 k[KP];
    f32x4 v[4][VP];
  };
  auto request = [&](Step& s, int at) {
#pragma unroll
    for (int p = 0; p < KP; ++p) {
      const char* row = kBase + (uint64_t)((unsigned)slots[at + (lane & 7) + 8 * (p & 1)] & 0x7fffffffu) * x.kStride;
      s.k[p] = *reinterpret_cast<const u32x4*>(row + kOff[p]);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const char* row = vBase + (uint64_t)((unsigned)slots[at + 4 * quad + i] & 0x7fffffffu) * x.vStride;
#pragma unroll
      for (int p = 0; p < VP; ++p) s.v[i][p] = *reinterpret_cast<const f32x4*>(row + vOff[p]);
    }
    __builtin_amdgcn_sched_barrier(0);  // nothing of the step before is touched (and waited for) ahead of these loads
  };
  // `own` in the lanes of `banks` (0xc: 8 .. 15 of each 16, 0x3: 0 .. 7) replaced by what the lane 8 aside has in `other`
  auto swapped = [](uint32_t own, uint32_t other, auto banks) {
    return (uint32_t)__builtin_amdgcn_update_dpp((int)own, (int)other, 0x128 /* rotate 16 lanes by 8 */, 0xf, decltype(banks)::value, false);
  };
  constexpr std::integral_constant<int, 0xc> kUpper{};
  constexpr std::integral_constant<int, 0x3> kLower{};

  f32x4 acc[NC][RUN];
  float most[NC], m[NC], mRef[NC], l[NC];  // the largest score, the same in units of log2, what scores are taken against, the sum
  auto clear = [&] {
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      most[c] = m[c] = -INFINITY, mRef[c] = l[c] = 0.f;
#pragma unroll
      for (int t = 0; t < RUN; ++t) acc[c][t] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
  };
  auto multiply = [&](Step& s, int at, bool all, auto withCare) {  // all: every one of the tokens counts
    constexpr bool CAREFUL = decltype(withCare)::value;
    u32x4 kf[KP];
#pragma unroll
    for (int p = 0; p < KP; ++p) {
#pragma unroll
      for (int w = 0; w < 4; ++w) kf[p][w] = p & 1 ? swapped(s.k[p][w], s.k[p - 1][w], kLower) : swapped(s.k[p][w], s.k[p + 1][w], kUpper);
      if (CAREFUL && 128 * (p >> 1) + 32 * quad + 16 * (p & 1) >= rowBytes) kf[p] = u32x4{0, 0, 0, 0};
    }
    bool counts[4] = {true, true, true, true};
    if (CAREFUL || !all) {
      const int4 m4 = *reinterpret_cast<const int4*>(slots + at + 4 * quad);
      counts[0] = m4.x >= 0, counts[1] = m4.y >= 0, counts[2] = m4.z >= 0, counts[3] = m4.w >= 0;
    }
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      f32x4 w = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int p = 0; p < KP; ++p)
#pragma unroll
        for (int e = 0; e < 4; ++e) w = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(kf[p][e]), qf[c][p][e], w, 0, 0, 0);
      if (CAREFUL || !all) {
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = counts[i] ? w[i] : -INFINITY;
      }
      float mt = fmaxf(fmaxf(w[0], w[1]), fmaxf(w[2], w[3]));
      if (__builtin_amdgcn_ballot_w64(mt > most[c]) != 0) {
        auto sw = __builtin_amdgcn_permlane32_swap(__float_as_uint(mt), __float_as_uint(mt), false, false);
        mt = fmaxf(__uint_as_float(sw[0]), __uint_as_float(sw[1]));
        sw = __builtin_amdgcn_permlane16_swap(__float_as_uint(mt), __float_as_uint(mt), false, false);
        mt = fmaxf(__uint_as_float(sw[0]), __uint_as_float(sw[1]));
        if (mt > most[c]) {
          most[c] = mt;
          const float mNew = mt * a.scaleLog2e;
          const float corr = m[c] == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m[c] - mNew);  // (no maximum yet: the sums are 0, or NaN)
          m[c] = mRef[c] = mNew;
          l[c] *= corr;
#pragma unroll
          for (int t = 0; t < RUN; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[c][t][i] *= corr;
        }
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        w[i] = __builtin_amdgcn_exp2f(CAREFUL ? behindRounded(w[i] * a.scaleLog2e, mRef[c]) : fmaf(w[i], a.scaleLog2e, -mRef[c]));
        l[c] += w[i];
      }
#pragma unroll
      for (int t = 0; t < RUN; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float vi = s.v[i][t / 4][t % 4];
          if constexpr (CAREFUL) {
            vi = counts[i] ? vi : 0.f;
            const bool finite = (__float_as_uint(vi) & 0x7f800000u) != 0x7f800000u;
            acc[c][t] = __builtin_amdgcn_mfma_f32_16x16x4f32(finite ? 0.f : vi, w[i] > 0.f ? 1.f : w[i], acc[c][t], 0, 0, 0);
            vi = finite ? vi : 0.f;
          }
          acc[c][t] = __builtin_amdgcn_mfma_f32_16x16x4f32(vi, w[i], acc[c][t], 0, 0, 0);
        }
    }
  };
  // the wave's share of a block, after the block's slots have been published
  auto walk = [&](int n, bool clean, auto withCare) {
    const int share = ((n + kPxWaves - 1) / kPxWaves + TOKENS - 1) / TOKENS * TOKENS;  // whole steps
    const int from = min(wave * share, kPxBlock - TOKENS), to = min(n, wave * share + share);
    const int last = from + (to - from - 1) / TOKENS * TOKENS;
    Step s0;
    request(s0, from);  // (also where the wave has no step: all of the block's slots can be read)
    if constexpr (decltype(withCare)::value) {
      for (int at = from; at < to; at += TOKENS) {
        multiply(s0, at, false, withCare);
        request(s0, min(at + TOKENS, last));
      }
    } else {
      Step s1;
      int at = from;
      // (the last one or two steps stand by themselves: a branch around the loads of the loop would make every wait one for all of them)
      for (; at + 2 * TOKENS < to; at += 2 * TOKENS) {
        request(s1, at + TOKENS);
        multiply(s0, at, clean, withCare);
        request(s0, at + 2 * TOKENS);
        multiply(s1, at + TOKENS, clean, withCare);
      }
      if (at + TOKENS < to) {
        request(s1, at + TOKENS);
        multiply(s0, at, clean, withCare);
        multiply(s1, at + TOKENS, clean && at + 2 * TOKENS <= n, withCare);
      } else if (at < to) {
        multiply(s0, at, clean && at + TOKENS <= n, withCare);
      }
    }
  };
  // Publishes the slots of [block, block + n): a thread looks up every 256th (past the last: that one again).
  auto publish = [&](int block, int n) {
    __syncthreads();  // every wave is done with the block before
    bool bad = false;
    for (int i = threadIdx.x; i < kPxBlock; i += kPxWaves * 64) {
      if (i >= n + kPxWaves * TOKENS) break;  // (no step reaches further)
      const int64_t slot = ldIndex(x.loc, block + min(i, n - 1), x.loc64);
      const bool in = slot >= 0 && slot < a.slots;  // slots outside the pool are skipped, never dereferenced
      slots[i] = in && i < n ? (int)slot : (int)((in ? (unsigned)slot : 0u) | 0x80000000u);
      bad |= !in;
    }
    const bool waveBad = __builtin_amdgcn_ballot_w64(bad) != 0;
    if (lane == 0) badBuf[wave] = waveBad;
    __syncthreads();
    return !(badBuf[0] | badBuf[1] | badBuf[2] | badBuf[3]);
  };

  clear();
  for (int block = begin; block < end; block += kPxBlock) {
    const int n = min(kPxBlock, end - block);
    const bool clean = publish(block, n);
    walk(n, clean, std::false_type{});
  }
  uint32_t largest = 0;
  bool far = false;
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    far |= pairOf[c] >= 0 && (pxFar(m[c]) || !(l[c] < INFINITY));  // (of scores far below the maximum l alone may have become too large)
#pragma unroll
    for (int t = 0; t < RUN; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) largest = max(largest, pairOf[c] >= 0 ? __float_as_uint(acc[c][t][i]) & 0x7fffffffu : 0u);
  }
  if (__syncthreads_or(far || largest >= 0x7f800000u)) {
    clear();
    for (int block = begin; block < end; block += kPxBlock) {
      const int n = min(kPxBlock, end - block);
      publish(block, n);
      walk(n, false, std::true_type{});
    }
  }

  // every lane group holds its own share of l; then waves 2 and 3 hand their sums to 0 and 1, and 1 its to 0
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    auto sw = __builtin_amdgcn_permlane32_swap(__float_as_uint(l[c]), __float_as_uint(l[c]), false, false);
    l[c] = __uint_as_float(sw[0]) + __uint_as_float(sw[1]);
    sw = __builtin_amdgcn_permlane16_swap(__float_as_uint(l[c]), __float_as_uint(l[c]), false, false);
    l[c] = __uint_as_float(sw[0]) + __uint_as_float(sw[1]);
    if (l[c] != l[c] && m[c] == -INFINITY) m[c] = 0.f;  // scores that are not numbers alone: as a maximum of minus infinity they would be left out
  }
#pragma unroll
  for (int givers = kPxWaves / 2; givers >= 1; givers >>= 1) {
    __syncthreads();
    if (wave >= givers && wave < 2 * givers) {
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        stateBuf[wave - givers][c][0][lane] = m[c], stateBuf[wave - givers][c][1][lane] = l[c];
#pragma unroll
        for (int t = 0; t < RUN; ++t) pxLds[((wave - givers) * NC * RUN + c * RUN + t) * 64 + lane] = acc[c][t];
      }
    }
    __syncthreads();
    if (wave < givers) {
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        const float m2 = stateBuf[wave][c][0][lane], l2 = stateBuf[wave][c][1][lane], mNew = fmaxf(m[c], m2);
        const float w1 = m[c] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m[c] - mNew), w2 = m2 == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m2 - mNew);
        m[c] = mNew, l[c] = l[c] * w1 + l2 * w2;
#pragma unroll
        for (int t = 0; t < RUN; ++t) {
          const f32x4 o = pxLds[(wave * NC * RUN + c * RUN + t) * 64 + lane];
#pragma unroll
          for (int i = 0; i < 4; ++i) acc[c][t][i] = acc[c][t][i] * w1 + o[i] * w2;
        }
      }
    }
  }
  if (wave != 0) return;
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    if (pairOf[c] < 0) continue;
    float* dst = partial + ((int64_t)pairOf[c] * x.nsplit + split) * (2 + a.d);
    if (quad == 0) dst[0] = m[c], dst[1] = l[c];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int t = 0; t < RUN; ++t) {
        const int e = S::place(4 * quad + i, t);
        if (e < a.d) dst[2 + e] = acc[c][t][i];
      }
  }
}

// ------------------------------------------------ 16-bit rows: shared by the waves through LDS --
// Eight waves share a stage of 64 tokens (32 of 512-byte rows): four groups of NC column tiles times two halves of the tokens, so a
// workgroup takes up to 192 columns from one read of a row. Rows go straight into a ring of stages in LDS (global_load_lds, 16 bytes
// to a lane, pieces XOR-swizzled by row), K is read as it lies, V through the transposing read; one barrier per stage. Against
// rows that each wave loads into its own registers, where V has to be turned round by lane permutations and a wave has a SIMD
// to itself (us, 16 000 tokens, bf16): 8 K/V heads of 128 with 192 columns each 99 -> 45, with 32 30.5 -> 27.9; 32 with 32 81.6 -> 65.7, with
// 12 66.5 -> 64.9 (5 us of each for a launch that merged them, which these no longer need; now, with one to four own tokens, 44.4, 27.0, 61.7
// and 60.6). Of the 36 us that 192 columns take in fp16,
// 11 do not grow with the prefix (slots, then rows; at the end 12.8 MB of partial results); in the others the two waves of a SIMD
// multiply at the same time and then both take exponentials (matrix pipe busy for 7.5 us, vector ALUs for 11, LDS between them). Half the
// waves a phase behind the other half was no faster (45 us).
//
// The maximum is followed when a score exceeds it by more than 2^8. bf16 probabilities are cut into three bf16 parts, all 24 bits of
// them (as the own tokens' kernels cut theirs; the third costs 1 to 9 %: 16001 tokens, 48 sequences of 4 columns each, all launches, 47.8 -> 51.8 us, 3 of them 28.6 ->
// 28.8). fp16 ones, times 2^7 (so at most 2^15), into two fp16 parts: 22 bits of those down to 2^-10 of the largest, 16 down
// to 2^-16, less than 2^-32 of the largest in any case (an argument of -10 is rounded to 2^-21 of its exponential before that); a
// step that has smaller ones multiplies what is left of them times 2^24, 2^48 ... too, until nothing is left.
constexpr int kPtWaves = 8;
constexpr float kPtRescaleStep = 8.f;  // log2 domain
constexpr float kPtTwoParts = 16.f;    // two fp16 parts hold 16 bits of what is at least 2^-this
template <typename T, int D>
struct PtShape {
  static constexpr int HALVES = D == 256 ? 1 : 2;                              // shares of a stage's tokens, 32 each
  static constexpr int TOKENS = 32 * HALVES, COLUMN_WAVES = kPtWaves / HALVES;
  static constexpr int ROWB = D * 2, CPR = ROWB / 16, RPL = 64 / CPR;         // pieces of a row, rows of a wave's load
  static constexpr int LOADS = TOKENS / RPL / kPtWaves;                        // of a wave, per matrix and stage
  static constexpr int STAGEB = 2 * TOKENS * ROWB, STAGES = 4;
  static constexpr int KS = D / 32, DT = D / 16;
  // XOR on the 16-byte piece index of row r: 16 rows' pieces of one index of K fall on 16 different bank groups, the 8 rows x 32
  // bytes of half a transposing read of V on 8
  static __device__ __forceinline__ int swizzleK(int r) { return D >= 128 ? (r & 15) : ((r >> 1) & 7); }
  static __device__ __forceinline__ int swizzleV(int r) { return D >= 128 ? 2 * (r & 7) : 2 * ((r >> 1) & 3); }
};
template <typename T>
struct PtMfma;
template <>
struct PtMfma<bf16_t> {
  typedef bf16x8 Frag;
  static __device__ __forceinline__ f32x4 run(u32x4 a, Frag b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), b, c, 0, 0, 0); }
  static constexpr float kRaise = 0.f;  // log2 of what probabilities are multiplied by
  static constexpr uint32_t kExponent = 0x7f80u;
};
template <>
struct PtMfma<half_t> {
  typedef f16x8 Frag;
  static __device__ __forceinline__ f32x4 run(u32x4 a, Frag b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), b, c, 0, 0, 0); }
  static constexpr float kRaise = 7.f;
  static constexpr uint32_t kExponent = 0x7c00u;
};
// The next part of eight numbers, and what it leaves. fp16: cut, not rounded, and subtracted in one mixed instruction each (half the
// instructions; what is left is then a number of up to 13 bits more, of which the second part, rounded, has 11).
template <typename T>
__device__ __forceinline__ typename PtMfma<T>::Frag ptPart(float (&x)[8]) {
  typename PtMfma<T>::Frag part;
#pragma unroll
  for (int i = 0; i < 8; i += 2) {
    if constexpr (std::is_same<T, half_t>::value) {
      typedef __fp16 Cut __attribute__((ext_vector_type(2)));
      typedef half_t Pair __attribute__((ext_vector_type(2)));
      const Cut cut = __builtin_amdgcn_cvt_pkrtz(x[i], x[i + 1]);
      const Pair pair = __builtin_bit_cast(Pair, cut);
      part[i] = pair[0], part[i + 1] = pair[1];
      float minus = -1.f;
      asm("" : "+s"(minus));  // (a constant here becomes a conversion and a subtraction)
      x[i] = fmaf(static_cast<float>(pair[0]), minus, x[i]), x[i + 1] = fmaf(static_cast<float>(pair[1]), minus, x[i + 1]);
    } else {
      part[i] = static_cast<T>(x[i]), part[i + 1] = static_cast<T>(x[i + 1]);
      x[i] -= static_cast<float>(part[i]), x[i + 1] -= static_cast<float>(part[i + 1]);
    }
  }
  return part;
}
template <typename T>
__device__ __forceinline__ typename PtMfma<T>::Frag ptLast(const float (&x)[8]) {  // eight numbers rounded
  typename PtMfma<T>::Frag part;
#pragma unroll
  for (int i = 0; i < 8; ++i) part[i] = static_cast<T>(x[i]);
  return part;
}

template <typename T, int D, int NC>
__global__ __launch_bounds__(kPtWaves * 64, 2) void decodePrefixTiledKernel(TaPrefixArgs x, float* __restrict__ partial) {
  using S = PtShape<T, D>;
  using M = PtMfma<T>;
  using Frag = typename M::Frag;
  constexpr int ROWB = S::ROWB, KS = S::KS, DT = S::DT, STAGES = S::STAGES, TOKENS = S::TOKENS, COLUMN_WAVES = S::COLUMN_WAVES;
  constexpr bool HALF = std::is_same<T, half_t>::value;
  const TaArgs& a = x.a;
  extern __shared__ __attribute__((aligned(16))) f32x4 ptLds[];  // the ring; at the end, sums on their way to the waves that add them up
  __shared__ __attribute__((aligned(16))) int slots[kPxBlock];  // of a block's tokens; negative: does not count
  __shared__ int badBuf[kPtWaves];
  __shared__ float stateBuf[S::HALVES == 2 ? COLUMN_WAVES : 1][NC][2][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 15, quad = lane >> 4;
  // (the second half's waves in the opposite order: waves i and i + 4 share a SIMD, and one of them may have a tile less)
  const int half = wave / COLUMN_WAVES, columnWave = half == 0 ? wave % COLUMN_WAVES : COLUMN_WAVES - 1 - wave % COLUMN_WAVES;

  // grid as in decodePrefixFloatKernel; tiles of columns are dealt out evenly, to the groups and to the waves of one: NC to a wave, or one
  // less (16 001 tokens, 192 columns: 36 us with two groups of 6 tiles, 40 us with full groups, one of 8 and one of 4)
  const int f = blockIdx.x, idx = f >> 3;
  const int perKv = a.heads / a.kvHeads, columns = a.batch * perKv, tiles = (columns + 15) / 16, groups = x.groups;
  const int group = idx % groups, u = (idx / groups) * 8 + (f & 7);
  if (u >= a.kvHeads * x.nsplit) return;  // the grid is rounded up to whole rounds of the XCDs
  const int kvh = u % a.kvHeads, split = u / a.kvHeads;
  const int begin = split * x.chunk, end = min(x.len, begin + x.chunk);
  const int groupTile = (int)((int64_t)group * tiles / groups), groupTiles = (int)((int64_t)(group + 1) * tiles / groups) - groupTile;
  const int firstTile = columnWave * groupTiles / COLUMN_WAVES, mine = (columnWave + 1) * groupTiles / COLUMN_WAVES - firstTile;
  const int firstColumn = (groupTile + firstTile) * 16;
  const bool active = NC > 1 || mine > 0;  // (a wave without columns only copies)

  Frag qf[NC][KS];
  int pairOf[NC];  // row of the partial results of this lane's column, or -1
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    const int column = firstColumn + c * 16 + col;
    const bool have = c < mine && column < columns;
    const int b = have ? column / perKv : 0, h = kvh * perKv + (have ? column % perKv : 0);
    pairOf[c] = have ? b * a.heads + h : -1;
    const T* src = reinterpret_cast<const T*>(a.q) + b * a.qBatchStride + h * a.qHeadStride;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      const int e = 32 * s + 8 * quad;
      u32x4 v = *reinterpret_cast<const u32x4*>(src + (e < a.d ? e : 0));
      if (!have || e >= a.d) v = u32x4{0, 0, 0, 0};
      qf[c][s] = __builtin_bit_cast(Frag, v);
    }
  }

  // copies: load i of this wave fills the KiB i * 8 + wave of a matrix; lane l owns the place (row l / CPR, piece l % CPR) of it and
  // fetches the piece that the swizzle puts there (pieces past the row's end repeat its first one)
  const unsigned ring = (unsigned)(uintptr_t)ptLds;
  const char* kSrc[S::LOADS];
  const char* vSrc[S::LOADS];
  int rowOf[S::LOADS];
#pragma unroll
  for (int i = 0; i < S::LOADS; ++i) {
    rowOf[i] = (i * kPtWaves + wave) * S::RPL + lane / S::CPR;
    const int p = lane % S::CPR, kc = (p ^ S::swizzleK(rowOf[i])) * 8, vc = (p ^ S::swizzleV(rowOf[i])) * 8;
    kSrc[i] = reinterpret_cast<const char*>(reinterpret_cast<const T*>(a.k) + kvh * a.kHeadStride + (kc < a.d ? kc : 0));
    vSrc[i] = reinterpret_cast<const char*>(reinterpret_cast<const T*>(a.v) + kvh * a.vHeadStride + (vc < a.d ? vc : 0));
  }
  auto copy = [&](int at, int stage) {
    const unsigned to = ring + (unsigned)(stage * S::STAGEB + wave * 1024);
#pragma unroll
    for (int i = 0; i < S::LOADS; ++i) {
      const uint64_t n = (unsigned)slots[at + rowOf[i]] & 0x7fffffffu;
      globalLoadToLds16(kSrc[i] + n * x.kStride, to + i * kPtWaves * 1024u);
      globalLoadToLds16(vSrc[i] + n * x.vStride, to + TOKENS * ROWB + i * kPtWaves * 1024u);
    }
  };

  f32x4 acc[NC][DT];
  float most[NC], m[NC], mRef[NC], l[NC];  // the largest score, the same in units of log2, what scores are taken against, the sum
  auto clear = [&] {
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      most[c] = m[c] = -INFINITY, mRef[c] = l[c] = 0.f;
#pragma unroll
      for (int t = 0; t < DT; ++t) acc[c][t] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
  };
  // What a stage goes through. Rows of K and of V are asked for ahead of what is done with those before them: the first products of
  // a stage find K in registers, those with V the first kAhead places.
  constexpr int kAhead = HALF && D == 128 && NC == 2 ? 2 : 4;  // (four would not fit the registers there)
  constexpr bool kAheadK = D < 256;  // (rows of 512 bytes: the registers for it are not there)
  typedef __attribute__((address_space(3))) const u32x4* LdsPiece;
  typedef __attribute__((address_space(3))) s16x4* LdsTr;
  auto readK = [&](u32x4 (&kf)[2][KS], int stage) {
    const unsigned at = ring + (unsigned)(stage * S::STAGEB + half * 32 * ROWB);
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        const int row = 16 * t + col;
        kf[t][s] = *(LdsPiece)(uintptr_t)(at + (unsigned)(row * ROWB + (((4 * s + quad) ^ S::swizzleK(row)) << 4)));
      }
  };
  auto scoresOf = [&](const u32x4 (&kf)[2][KS], f32x4 (&s4)[NC][2], auto columnTiles, auto withCare) {
    constexpr int N = decltype(columnTiles)::value;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
#pragma unroll
      for (int c = 0; c < N; ++c) s4[c][t] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
#pragma unroll
    for (int s = 0; s < KS; ++s)
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        u32x4 k = kf[t][s];
        if (decltype(withCare)::value && 32 * s + 8 * quad >= a.d) k = u32x4{0, 0, 0, 0};  // (an infinity against q's zeros would be NaN)
#pragma unroll
        for (int c = 0; c < N; ++c) s4[c][t] = M::run(k, qf[c][s], s4[c][t]);
      }
  };
  struct Counts {  // which of the lane's eight tokens count
    bool of[8];
  };
  auto countsOf = [&](int at, bool all) {
    Counts n;
#pragma unroll
    for (int i = 0; i < 8; ++i) n.of[i] = true;
    if (!all) {
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const int4 m4 = *reinterpret_cast<const int4*>(slots + at + 32 * half + 16 * t + 4 * quad);
        n.of[4 * t] = m4.x >= 0, n.of[4 * t + 1] = m4.y >= 0, n.of[4 * t + 2] = m4.z >= 0, n.of[4 * t + 3] = m4.w >= 0;
      }
    }
    return n;
  };
  // the scores of column tile c: its maximum followed (and all that was summed against the old one), as powers of two
  auto powersOf = [&](int c, const f32x4 (&s4)[2], const Counts& n, bool all, float (&arg)[8], bool follow, float step, auto withCare) {
#pragma unroll
    for (int i = 0; i < 8; ++i) arg[i] = s4[i >> 2][i & 3];
    if (!all) {
#pragma unroll
      for (int i = 0; i < 8; ++i) arg[i] = n.of[i] ? arg[i] : -INFINITY;
    }
    if (follow) {
      float mt = arg[0];
#pragma unroll
      for (int i = 1; i < 8; ++i) mt = fmaxf(mt, arg[i]);
      if (__builtin_amdgcn_ballot_w64(mt * a.scaleLog2e > m[c] + step) != 0) {
        auto sw = __builtin_amdgcn_permlane32_swap(__float_as_uint(mt), __float_as_uint(mt), false, false);
        mt = fmaxf(__uint_as_float(sw[0]), __uint_as_float(sw[1]));
        sw = __builtin_amdgcn_permlane16_swap(__float_as_uint(mt), __float_as_uint(mt), false, false);
        mt = fmaxf(__uint_as_float(sw[0]), __uint_as_float(sw[1]));
        if (mt > most[c]) {
          most[c] = mt;
          const float mNew = mt * a.scaleLog2e;
          const float corr = m[c] == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m[c] - mNew);  // (no maximum yet: the sums are 0, or NaN)
          m[c] = mRef[c] = mNew;
          l[c] *= corr;
#pragma unroll
          for (int t = 0; t < DT; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[c][t][i] *= corr;
        }
      }
    }
    const float ref = mRef[c] - M::kRaise;
#pragma unroll
    for (int i = 0; i < 8; ++i) arg[i] = decltype(withCare)::value ? behindRounded(arg[i] * a.scaleLog2e, ref) : fmaf(arg[i], a.scaleLog2e, -ref);
  };
  auto readV = [&](int d, int stage) {  // eight tokens at the lane's place of the head
    const unsigned at = ring + (unsigned)(stage * S::STAGEB + (TOKENS + half * 32) * ROWB);
    const int vRow = 4 * quad + ((lane & 15) >> 2);
    u32x2 v[2];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const int row = 16 * t + vRow;
      const unsigned piece = (unsigned)((2 * d + ((lane & 3) >> 1)) ^ S::swizzleV(row)) << 4;
      v[t] = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsTr)(uintptr_t)(at + (unsigned)(row * ROWB + (lane & 1) * 8) + piece)));
    }
    return u32x4{v[0][0], v[0][1], v[1][0], v[1][1]};
  };
  auto infinite = [](u32x4 v) {  // ones where V is not finite
    u32x4 bad;
#pragma unroll
    for (int j = 0; j < 4; ++j)
      bad[j] = ((v[j] & M::kExponent) == M::kExponent ? 0xffffu : 0u) | ((v[j] & (M::kExponent << 16)) == (M::kExponent << 16) ? 0xffff0000u : 0u);
    return bad;
  };
  auto keepOf = [&](const Counts& n) {  // ones where a token counts
    u32x4 keep = {~0u, ~0u, ~0u, ~0u};
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (!n.of[i]) keep[i >> 1] &= i & 1 ? 0xffffu : 0xffff0000u;
    return keep;
  };
  // What two parts leave of probabilities, times 2^24, 2^48 ... (the scores once more: keeping them for
  // this would cost the registers of a column tile).
  auto addRest = [&](int stage, int at, bool all, auto columnTiles, auto withCare) {
    constexpr bool CAREFUL = decltype(withCare)::value;
    constexpr int N = decltype(columnTiles)::value;
    const Counts n = countsOf(at, all);
    const u32x4 keep = keepOf(n);
    u32x4 kf[2][KS];
    readK(kf, stage);
    f32x4 s4[NC][2];
    scoresOf(kf, s4, columnTiles, withCare);
#pragma unroll
    for (int c = 0; c < N; ++c) {
      float w[8];
      powersOf(c, s4[c], n, all, w, false, 0.f, withCare);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        w[i] = __builtin_amdgcn_exp2f(w[i]);
        w[i] = w[i] == w[i] ? w[i] : 0.f;  // (NaN is in the first part)
      }
      auto leave = [&] {  // the first part, and the second
        const Frag first = ptPart<T>(w), second = ptLast<T>(w);
#pragma unroll
        for (int i = 0; i < 8; ++i) w[i] -= static_cast<float>(second[i]);
        return std::pair<Frag, Frag>{first, second};
      };
      leave();
      float back = 1.f;
      for (int round = 0; round < 6; ++round) {  // (2^-169 is all that could be left after them)
        bool any = false;
        back *= 0x1p-24f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          w[i] *= 0x1p24f;
          any |= w[i] != 0.f;
        }
        if (__builtin_amdgcn_ballot_w64(any) == 0) break;
        const auto [hi, lo] = leave();
#pragma unroll
        for (int d = 0; d < DT; ++d) {
          u32x4 v = readV(d, stage);
          if constexpr (CAREFUL) v &= keep & ~infinite(v);
          f32x4 rest = M::run(v, hi, f32x4{0.f, 0.f, 0.f, 0.f});
          rest = M::run(v, lo, rest);
#pragma unroll
          for (int i = 0; i < 4; ++i) acc[c][d][i] += rest[i] * back;
        }
      }
    }
  };
  // the stages of a block, after its slots have been published; clean: all of its slots lie in the pool
  auto walk = [&](int n, bool clean, auto columnTiles, auto withCare) {
    constexpr bool CAREFUL = decltype(withCare)::value;
    constexpr int N = decltype(columnTiles)::value;
    const int stages = (n + TOKENS - 1) / TOKENS;
    // this wave's copies of a stage have landed (loads end in order; `behind` stages are on their way) and then everybody's have
    auto landed = [&](bool behind) {
      constexpr int kBehind = 2 * S::LOADS * (STAGES - 3);
      if (behind) __builtin_amdgcn_s_waitcnt(0x0f70 | (kBehind & 15) | (kBehind >> 4) << 14);
      else __builtin_amdgcn_s_waitcnt(0x0f70);
      asm volatile("" : : : "memory");
      __builtin_amdgcn_s_barrier();
      asm volatile("" : : : "memory");
    };
#pragma unroll
    for (int s = 0; s < STAGES - 1; ++s)
      if (s < stages) copy(s * TOKENS, s);
    __builtin_amdgcn_s_waitcnt(0x0f70);
    asm volatile("" : : : "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" : : : "memory");
    u32x4 kf[2][KS];
    if (kAheadK && active) readK(kf, 0);
    int stage = 0;
    for (int s = 0; s < stages; ++s) {
      const bool all = !CAREFUL && clean && (s + 1) * TOKENS <= n;
      const int next = stage + 1 == STAGES ? 0 : stage + 1;
      Frag hi[NC], lo[NC], last[HALF ? 1 : NC], some[CAREFUL ? NC : 1];
      u32x4 v[kAhead], keep = {~0u, ~0u, ~0u, ~0u};
      bool small = false;  // of a probability some bits may be left
      if (active) {
        f32x4 s4[NC][2];
        if (!kAheadK) readK(kf, stage);
        scoresOf(kf, s4, columnTiles, withCare);
        const Counts counts = countsOf(s * TOKENS, all);
        if constexpr (CAREFUL) keep = keepOf(counts);
#pragma unroll
        for (int d = 0; d < kAhead; ++d) v[d] = readV(d, stage);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int c = 0; c < N; ++c) {
          float w[8], lowest = 0.f;
          powersOf(c, s4[c], counts, all, w, true, CAREFUL ? 0.f : kPtRescaleStep, withCare);
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            if (HALF) lowest = fminf(lowest, w[i]);
            w[i] = __builtin_amdgcn_exp2f(w[i]);
            l[c] += w[i];
          }
          small |= lowest < M::kRaise - kPtTwoParts;
          if constexpr (CAREFUL) {
#pragma unroll
            for (int i = 0; i < 8; ++i) some[c][i] = static_cast<T>(w[i] > 0.f ? 1.f : w[i]);
          }
          hi[c] = ptPart<T>(w);
          if constexpr (HALF) lo[c] = ptLast<T>(w);
          else lo[c] = ptPart<T>(w), last[c] = ptLast<T>(w);
        }
      }
      if (s + 1 < stages) {
        landed(s + STAGES - 2 < stages);
        // (everybody has read the stage before this one: its place is free)
        if (s + STAGES - 1 < stages) copy((s + STAGES - 1) * TOKENS, stage == 0 ? STAGES - 1 : stage - 1);
        if (kAheadK && active) readK(kf, next);
        __builtin_amdgcn_sched_barrier(0);
      }
      if (active) {
#pragma unroll
        for (int d = 0; d < DT; ++d) {
          u32x4 now = v[d % kAhead];
          if (d + kAhead < DT) v[d % kAhead] = readV(d + kAhead, stage);
          if constexpr (CAREFUL) {
            now &= keep;
            const u32x4 bad = infinite(now), odd = now & bad;
            now &= ~bad;
#pragma unroll
            for (int c = 0; c < N; ++c) acc[c][d] = M::run(odd, some[c], acc[c][d]);
          }
#pragma unroll
          for (int c = 0; c < N; ++c) acc[c][d] = M::run(now, hi[c], acc[c][d]);
#pragma unroll
          for (int c = 0; c < N; ++c) acc[c][d] = M::run(now, lo[c], acc[c][d]);
          if constexpr (!HALF) {
#pragma unroll
            for (int c = 0; c < N; ++c) acc[c][d] = M::run(now, last[c], acc[c][d]);
          }
        }
        if constexpr (HALF) {
          if (__builtin_amdgcn_ballot_w64(small) != 0) addRest(stage, s * TOKENS, all, columnTiles, withCare);
        }
      }
      stage = next;
    }
  };
  // Publishes the slots of [block, block + n) (up to a whole stage: that of the last token again).
  auto publish = [&](int block, int n) {
    __syncthreads();  // every wave is done with the block before
    bool bad = false;
    for (int i = threadIdx.x; i < (n + TOKENS - 1) / TOKENS * TOKENS; i += kPtWaves * 64) {
      const int64_t slot = ldIndex(x.loc, block + min(i, n - 1), x.loc64);
      const bool in = slot >= 0 && slot < a.slots;  // slots outside the pool are skipped, never dereferenced
      slots[i] = in && i < n ? (int)slot : (int)((in ? (unsigned)slot : 0u) | 0x80000000u);
      bad |= !in;
    }
    const bool waveBad = __builtin_amdgcn_ballot_w64(bad) != 0;
    if (lane == 0) badBuf[wave] = waveBad;
    __syncthreads();
    bool any = false;
#pragma unroll
    for (int w = 0; w < kPtWaves; ++w) any |= badBuf[w] != 0;
    return !any;
  };

  clear();
  for (int block = begin; block < end; block += kPxBlock) {
    const int n = min(kPxBlock, end - block);
    const bool clean = publish(block, n);
    if (NC == 1 || mine == NC) walk(n, clean, std::integral_constant<int, NC>{}, std::false_type{});
    else walk(n, clean, std::integral_constant<int, NC == 1 ? 1 : NC - 1>{}, std::false_type{});
  }
  uint32_t largest = 0;
  bool far = false;
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    far |= pairOf[c] >= 0 && (pxFar(m[c]) || !(l[c] < INFINITY));  // (as in decodePrefixFloatKernel)
#pragma unroll
    for (int t = 0; t < DT; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) largest = max(largest, pairOf[c] >= 0 ? __float_as_uint(acc[c][t][i]) & 0x7fffffffu : 0u);
  }
  if (__syncthreads_or(far || largest >= 0x7f800000u)) {
    clear();
    for (int block = begin; block < end; block += kPxBlock) {
      const int n = min(kPxBlock, end - block);
      publish(block, n);
      walk(n, false, std::integral_constant<int, NC>{}, std::true_type{});
    }
  }

  // every lane group holds its own share of l; the waves of the second half hand their sums to those of the first
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    auto sw = __builtin_amdgcn_permlane32_swap(__float_as_uint(l[c]), __float_as_uint(l[c]), false, false);
    l[c] = __uint_as_float(sw[0]) + __uint_as_float(sw[1]);
    sw = __builtin_amdgcn_permlane16_swap(__float_as_uint(l[c]), __float_as_uint(l[c]), false, false);
    l[c] = __uint_as_float(sw[0]) + __uint_as_float(sw[1]);
    if (l[c] != l[c] && m[c] == -INFINITY) m[c] = 0.f;  // scores that are not numbers alone: as a maximum of minus infinity they would be left out
  }
  if constexpr (S::HALVES == 2) __syncthreads();
  if (half == 1) {
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      stateBuf[columnWave][c][0][lane] = m[c], stateBuf[columnWave][c][1][lane] = l[c];
#pragma unroll
      for (int t = 0; t < DT; ++t) ptLds[((columnWave * NC + c) * DT + t) * 64 + lane] = acc[c][t];
    }
  }
  if constexpr (S::HALVES == 2) __syncthreads();
  if (half == 1) return;
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    float mNew = m[c], w1 = 1.f, w2 = 0.f, sum = l[c];
    if constexpr (S::HALVES == 2) {
      const float m2 = stateBuf[columnWave][c][0][lane];
      mNew = fmaxf(m[c], m2);
      w1 = m[c] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m[c] - mNew), w2 = m2 == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m2 - mNew);
      sum = l[c] * w1 + stateBuf[columnWave][c][1][lane] * w2;
    }
    float* dst = partial + ((int64_t)pairOf[c] * x.nsplit + split) * (2 + a.d);
    if (pairOf[c] < 0) continue;
    // (sums are against the maximum less the raise)
    if (quad == 0) *reinterpret_cast<float2*>(dst) = float2{mNew - M::kRaise, sum};
#pragma unroll
    for (int t = 0; t < DT; ++t) {
      const int e = 16 * t + 4 * quad;
      if (e >= a.d) continue;
      f32x4 r = acc[c][t];
      if constexpr (S::HALVES == 2) {
        const f32x4 o = ptLds[((columnWave * NC + c) * DT + t) * 64 + lane];
#pragma unroll
        for (int i = 0; i < 4; ++i) r[i] = r[i] * w1 + o[i] * w2;
      }
      *reinterpret_cast<float2*>(dst + 2 + e) = float2{r[0], r[1]};
      *reinterpret_cast<float2*>(dst + 4 + e) = float2{r[2], r[3]};
    }
  }
}

// out[b, h, :] from the partial results of the prefix's chunks and of the sequence's own (see mergeChunks), WAVES to a (sequence,
// head): every wave works out the weights of all shares, lane s those of shares s, s + 64, ..., then takes every WAVES-th share. The
// length, the (maximum, sum) pairs and the first shares' elements are asked for before any of them is waited for; rows of shares
// without tokens were never written, and what is read from them is discarded by a select.
template <typename T, int WAVES>
__global__ __launch_bounds__(256) void decodePrefixMergeKernel(T* __restrict__ out, const float* __restrict__ shared, int nShared, const float* __restrict__ own,
                                                               int nOwn, int chunk, float raise, const void* bLen, bool len64, int maxLen, int walked, int64_t pairs, int heads, int d) {
  constexpr int kBatch = 9, kMaxPerLane = 4, kPerLane = 8;  // 256 elements of a row (those from 256 blockIdx.y on), at most 512 shares
  __shared__ float red[4][64 * kMaxPerLane];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, part = wave % WAVES;
  const int64_t pair = (int64_t)blockIdx.x * (4 / WAVES) + wave / WAVES;
  if (WAVES == 1 && pair >= pairs) return;
  const int row = 2 + d, all = nShared + nOwn, first = 256 * blockIdx.y;
  const float* const sharedRows = shared + pair * nShared * row;
  const float* const ownRows = own + pair * nOwn * row;
  auto rowOf = [&](int s) { return s < nShared ? sharedRows + (int64_t)s * row : ownRows + (int64_t)(s - nShared) * row; };
  float ms[kPerLane], ls[kPerLane], v[kBatch][kMaxPerLane];
#pragma unroll
  for (int k = 0; k < kPerLane; ++k) {
    if (64 * k >= all) break;
    const float* r = rowOf(min(lane + 64 * k, all - 1));
    ms[k] = r[0] - (lane + 64 * k < nShared ? 0.f : raise), ls[k] = r[1];
  }
  auto loadBatch = [&](int s0) {
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      const float* r = rowOf(min(s0 + WAVES * u, all - 1)) + 2;
#pragma unroll
      for (int k = 0; k < kMaxPerLane; ++k) {
        const int e = first + lane + 64 * k;
        v[u][k] = e < d ? r[e] : 0.f;
      }
    }
  };
  loadBatch(part);
  const int used = nShared + (nOwn == 0 ? 0 : chunksWritten(walked + cutLength(bLen, pair / heads, len64, maxLen), chunk));
  float m = -INFINITY;
#pragma unroll
  for (int k = 0; k < kPerLane; ++k) {
    if (64 * k >= all) break;
    if (lane + 64 * k >= used) ms[k] = -INFINITY, ls[k] = 0.f;
    m = fmaxf(m, ms[k]);
  }
  m = waveMax(m);
  float sum = 0.f;
#pragma unroll
  for (int k = 0; k < kPerLane; ++k) {
    if (64 * k >= all) break;
    ms[k] = ms[k] == -INFINITY ? 0.f : exp2f(ms[k] - m);  // the weight
    sum += ls[k] * ms[k];
  }
  const float total = waveSum(sum), inv = total == 0.f ? 0.f : 1.f / total;
  float acc[kMaxPerLane] = {0.f, 0.f, 0.f, 0.f};
  for (int s0 = part; s0 < used; s0 += WAVES * kBatch) {
    if (s0 != part) loadBatch(s0);
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      const int s = s0 + WAVES * u, owner = min(s, all - 1) >> 6;  // wave-uniform
      float w = 0.f;
#pragma unroll
      for (int k = 0; k < kPerLane; ++k) {
        if (64 * k >= all) break;
        w = owner == k ? ms[k] : w;
      }
      w = __shfl(w, s & 63, 64) * inv;
#pragma unroll
      for (int k = 0; k < kMaxPerLane; ++k) acc[k] += s < used ? w * v[u][k] : 0.f;
    }
  }
  if (WAVES == 1) {
#pragma unroll
    for (int k = 0; k < kMaxPerLane; ++k) {
      const int e = first + lane + 64 * k;
      if (e < d) out[pair * d + e] = static_cast<T>(acc[k]);
    }
    return;
  }
#pragma unroll
  for (int k = 0; k < kMaxPerLane; ++k) red[wave][lane + 64 * k] = acc[k];
  __syncthreads();
  if (wave == 0) {
#pragma unroll
    for (int k = 0; k < kMaxPerLane; ++k) {
      const int i = lane + 64 * k, e = first + i;
      if (e < d) out[pair * d + e] = static_cast<T>(red[0][i] + red[1][i] + red[2][i] + red[3][i]);
    }
  }
}

// ---------------------------------------------------------------- host side --
template <typename T, int D, int NC>
static diopiError_t launchTiled(hipStream_t stream, const TaPrefixArgs& x, int64_t wgs, float* partial) {
  const int lds = PtShape<T, D>::STAGES * PtShape<T, D>::STAGEB;
  static_assert(PtShape<T, D>::HALVES == 1 || PtShape<T, D>::STAGES * PtShape<T, D>::STAGEB >= PtShape<T, D>::COLUMN_WAVES * NC * PtShape<T, D>::DT * 64 * (int)sizeof(f32x4), "the sums of half the waves take the place of the ring");
  AMD_HIP(allowDynamicLds(reinterpret_cast<const void*>(decodePrefixTiledKernel<T, D, NC>), lds));
  hipLaunchKernelGGL((decodePrefixTiledKernel<T, D, NC>), dim3((unsigned)wgs), dim3(kPtWaves * 64), lds, stream, x, partial);
  AMD_LAUNCH_CHECK();
  return diopiSuccess;
}

template <int D, int NC>
static diopiError_t launchFloat(hipStream_t stream, const TaPrefixArgs& x, int64_t wgs, float* partial) {
  const int lds = kPxWaves / 2 * NC * PxShape<D>::RUN * 64 * (int)sizeof(f32x4);
  AMD_HIP(allowDynamicLds(reinterpret_cast<const void*>(decodePrefixFloatKernel<D, NC>), lds));
  hipLaunchKernelGGL((decodePrefixFloatKernel<D, NC>), dim3((unsigned)wgs), dim3(kPxWaves * 64), lds, stream, x, partial);
  AMD_LAUNCH_CHECK();
  return diopiSuccess;
}

diopiError_t mergeShares(hipStream_t stream, const TaArgs& a, diopiDtype_t dtype, void* out, const float* shared, int nShared, const TaPartials& own, int walked) {
  const int64_t pairs = (int64_t)a.batch * a.heads;
  // A wave has the elements of nine shares on their way at once. Up to those it needs no help; twice as many are still better left to
  // one than to four where there are many pairs: 2048 pairs, 10 shares 23.7 us (all launches) and 27.3; 512 pairs, 18 shares
  // 18.9 and 17.5.
  const int shares = nShared + own.nsplit;
  const bool narrow = shares <= 9 || (shares <= 18 && pairs >= 1024);
  const unsigned blocks = (unsigned)ceilDiv(a.d, 256);
#define PREFIX_MERGE(T)                                                                                                                               \
  do {                                                                                                                                                \
    if (narrow)                                                                                                                                       \
      hipLaunchKernelGGL((decodePrefixMergeKernel<T, 1>), dim3((unsigned)ceilDiv(pairs, 4), blocks), dim3(256), 0, stream, static_cast<T*>(out), shared, \
                         nShared, own.partial, own.nsplit, own.chunk, own.raise, a.bLen, a.len64, a.maxLen, walked, pairs, a.heads, a.d);            \
    else                                                                                                                                              \
      hipLaunchKernelGGL((decodePrefixMergeKernel<T, 4>), dim3((unsigned)pairs, blocks), dim3(256), 0, stream, static_cast<T*>(out), shared, nShared, \
                         own.partial, own.nsplit, own.chunk, own.raise, a.bLen, a.len64, a.maxLen, walked, pairs, a.heads, a.d);                      \
  } while (0)
  if (dtype == diopi_dtype_bfloat16) PREFIX_MERGE(bf16_t);
  else if (dtype == diopi_dtype_float16) PREFIX_MERGE(half_t);
  else PREFIX_MERGE(float);
#undef PREFIX_MERGE
  AMD_LAUNCH_CHECK();
  return diopiSuccess;
}

static diopiError_t decodeSharedPrefix(diopiContextHandle_t ctx, hipStream_t stream, TaPrefixArgs x, diopiDtype_t dtype, void* out) {
  TaArgs& a = x.a;
  const int64_t perKv = a.heads / a.kvHeads, columns = a.batch * perKv, cus = computeUnits(), itemsize = dtypeSize(dtype);
  const int D = a.d <= 64 ? 64 : a.d <= 128 ? 128 : 256;
  x.kStride = (unsigned)(a.kSlotStride * itemsize), x.vStride = (unsigned)(a.vSlotStride * itemsize);
  const bool tiled = itemsize == 2;
  const int64_t pairs = (int64_t)a.batch * a.heads, tiles = ceilDiv(columns, 16);
  const int64_t columnWaves = !tiled ? 1 : D == 256 ? PtShape<half_t, 256>::COLUMN_WAVES : PtShape<half_t, 128>::COLUMN_WAVES;
  const int ncMost = tiled ? (D == 256 ? 1 : D == 128 ? 2 : 3) : columns > 16 && D == 64 ? 2 : 1;  // (more spill registers)
  // The shortest chunk. Short ones keep more compute units busy, but every pair (sequence, head) has a partial result for each of
  // them, so it is 64 tokens while that leaves 16 of them for up to 256 pairs and fewer for more, 4 from 1024 on, and longer then,
  // up to 256. Heads of 128, us with this rule and with 256: 250 tokens, 32 heads, 16 sequences 10.0, 12.0, 500 11.1, 12.2; 32 on 8,
  // 48 sequences, 250 tokens 12.8, 15.9, 500 13.9, 15.8; with 64 for any number of pairs 2000 tokens would take the last 19.6, so 17.1. 32
  // chunks for few pairs: 4 sequences, 2000 tokens, 8 heads on 1 15.4, so 13.9; 32 on 8 14.1, so 13.1.
  const int64_t most = std::min<int64_t>(16, std::max<int64_t>(4, 4096 / pairs));
  const int64_t shortest = std::min<int64_t>(256, std::max<int64_t>(64, ceilDiv(x.len, most)));
  // Few groups of columns read a row least often, but where they and chunks as short as pays leave compute units without work, more
  // take it (8 K/V heads of 64, 192 columns each: 700 tokens 12.0 us, with the fewest groups 16.6; 4096 tokens 16.7 and 20.9 us).
  const int64_t fewest = ceilDiv(tiles, columnWaves * ncMost);
  const int64_t groups = std::max(fewest, std::min(ceilDiv(tiles, columnWaves), cus / (a.kvHeads * ceilDiv(x.len, shortest))));
  const int nc = (int)ceilDiv(ceilDiv(tiles, groups), columnWaves);
  x.groups = (int)groups;
  const int64_t step = tiled && D == 256 ? 32 : 64;  // of all waves
  const int64_t chunk = std::max({shortest, ceilDiv((int64_t)x.len * a.kvHeads * groups, cus), ceilDiv(x.len, kPxMaxSplit)});
  x.chunk = (int)(ceilDiv(chunk, step) * step);
  x.nsplit = (int)ceilDiv(x.len, x.chunk);
  const int64_t wgs = ceilDiv((int64_t)a.kvHeads * x.nsplit, 8) * 8 * groups;
  // (fewer than 2^32 threads to a launch)
  AMD_CHECK(wgs < 1 << 23 && pairs < 1 << 24, "shared prefix attention: %d sequences of %d heads exceed the grid limits", a.batch, a.heads);
  void* ws = nullptr;
  AMD_TRY(requireWorkspace(ctx, pairs * x.nsplit * (2 + a.d) * (int64_t)sizeof(float), &ws));
  float* partial = static_cast<float*>(ws);
#define TILED_CALL(T, SIZE, N) AMD_TRY((launchTiled<T, SIZE, N>(stream, x, wgs, partial)))
#define TILED_COLUMNS(T, SIZE) \
  do { if (nc == 1) TILED_CALL(T, SIZE, 1); else TILED_CALL(T, SIZE, 2); } while (0)
#define TILED_SIZES(T)                        \
  do {                                        \
    if (D == 64 && nc == 3) TILED_CALL(T, 64, 3); \
    else if (D == 64) TILED_COLUMNS(T, 64);       \
    else if (D == 128) TILED_COLUMNS(T, 128);     \
    else TILED_CALL(T, 256, 1);               \
  } while (0)
  if (tiled) {
    if (dtype == diopi_dtype_bfloat16) TILED_SIZES(bf16_t);
    else TILED_SIZES(half_t);
  } else if (D == 64) {
    AMD_TRY((nc == 1 ? launchFloat<64, 1> : launchFloat<64, 2>)(stream, x, wgs, partial));
  } else {
    AMD_TRY((D == 128 ? launchFloat<128, 1> : launchFloat<256, 1>)(stream, x, wgs, partial));
  }
#undef TILED_SIZES
#undef TILED_COLUMNS
#undef TILED_CALL
  TaPartials own{nullptr, 0, 1, 0.f};
  if (a.generic) {  // (rows of more than 512 bytes)
    TaAnyArgs any{};
    any.a = a;
    AMD_TRY(walkAny(ctx, stream, any, dtype, out, false, &own));
  } else {
    a.shared = partial, a.nShared = x.nsplit;
    AMD_TRY(decodePartials(ctx, stream, a, dtype, a.maxLen, out, &own));
    if (own.nsplit == 0) return diopiSuccess;
  }
  return mergeShares(stream, a, dtype, out, partial, x.nsplit, own, 0);
}

}  // namespace amd

using namespace amd;

extern "C" __attribute__((visibility("default"))) diopiError_t diopiTokenDecodeAttentionSharedPrefixInference(
    diopiContextHandle_t ctx, diopiTensorHandle_t outH, diopiConstTensorHandle_t qH, diopiConstTensorHandle_t kH,
    diopiConstTensorHandle_t vH, diopiConstTensorHandle_t prefixLocH, diopiConstTensorHandle_t locH,
    diopiConstTensorHandle_t startH, diopiConstTensorHandle_t lenH, int maxInputLen) {
  hipStream_t stream;
  AMD_TRY(getStream(ctx, &stream));
  TaViews t;
  TensorView out, prefix, densePrefix;
  AMD_TRY(getView(outH, &out, "out"));
  AMD_TRY(getView(qH, &t.q, "q"));
  AMD_TRY(getView(kH, &t.k, "k"));
  AMD_TRY(getView(vH, &t.v, "v"));
  AMD_TRY(getView(prefixLocH, &prefix, "prefix_loc"));
  AMD_TRY(getView(locH, &t.loc, "b_loc"));
  AMD_TRY(getView(startH, &t.start, "b_start_loc"));
  AMD_TRY(getView(lenH, &t.len, "b_seq_len"));
  TaPrefixArgs x;
  TaArgs& a = x.a;
  AMD_TRY(fillArgs(t, true, true, maxInputLen, &a));
  AMD_CHECK(prefix.defined() && prefix.ndim == 1, "shared prefix attention: prefix_loc must be a tensor of one dim");
  AMD_CHECK(prefix.dtype == diopi_dtype_int32 || prefix.dtype == diopi_dtype_int64, "shared prefix attention: prefix_loc must be int32 or int64, got %s",
            dtypeName(prefix.dtype));
  AMD_CHECK(prefix.shape[0] + (int64_t)maxInputLen <= 1 << 30, "shared prefix attention: %ld shared tokens and %d own ones exceed 2^30",
            (long)prefix.shape[0], maxInputLen);
  AMD_CHECK(out.defined() && out.dtype == t.q.dtype && out.ndim == 3 && out.isContiguous(), "shared prefix attention: out must be a dense tensor shaped like q");
  for (int d = 0; d < 3; ++d) AMD_CHECK(out.shape[d] == t.q.shape[d], "shared prefix attention: out must be shaped like q");
  if (t.q.numel == 0) return diopiSuccess;
  AMD_CHECK(a.batch <= 65535, "shared prefix attention: batch %d exceeds the grid limits", a.batch);
  AMD_CHECK(t.q.shape[2] <= kTaGenericMaxD, "shared prefix attention: head_dim %ld exceeds %d", (long)t.q.shape[2], kTaGenericMaxD);
  if (prefix.shape[0] == 0) return diopiTokenDecodeAttentionInference(ctx, outH, qH, kH, vH, locH, startH, lenH, maxInputLen);  // nothing is shared
  AMD_TRY(makeContiguous(ctx, stream, prefix, &densePrefix));
  x.loc = densePrefix.data, x.loc64 = prefix.dtype == diopi_dtype_int64, x.len = (int)prefix.shape[0];
  // head rows of whole 16-byte pieces up to 256 elements, slot numbers in 31 bits: the matrix pipe
  const int64_t bits = (int64_t)reinterpret_cast<uintptr_t>(a.k) | (int64_t)reinterpret_cast<uintptr_t>(a.v) |
                       (a.kSlotStride | a.kHeadStride | a.vSlotStride | a.vHeadStride | a.d) * t.q.itemsize;
  if ((bits & 15) == 0 && a.d <= 256 && a.slots <= 0x7fffffff && std::max(a.kSlotStride, a.vSlotStride) * t.q.itemsize <= 0xffffffffll) {
    if (!t.q.aligned16() || ((a.qBatchStride | a.qHeadStride) * t.q.itemsize) % 16 != 0) {  // a dense copy of q
      diopiTensorHandle_t th = nullptr;
      TensorView dense;
      AMD_TRY(requireTensor(ctx, t.q.shape, t.q.ndim, t.q.dtype, &th, &dense));
      AMD_TRY(stridedCopy(stream, t.q, dense));
      t.q = dense;
      AMD_TRY(fillArgs(t, true, true, maxInputLen, &a));
    }
    return decodeSharedPrefix(ctx, stream, x, t.q.dtype, out.data);
  }
  TaAnyArgs any{};
  any.a = a, any.loc = x.loc, any.locIs64 = x.loc64, any.walked = x.len;
  TaPartials own;
  AMD_TRY(walkAny(ctx, stream, any, t.q.dtype, out.data, true, &own));
  return own.nsplit == 0 ? diopiSuccess : mergeShares(stream, a, t.q.dtype, out.data, nullptr, 0, own, any.walked);
}
