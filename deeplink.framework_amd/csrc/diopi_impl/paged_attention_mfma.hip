// Attention of new tokens over a paged pool on the matrix pipe (see paged_attention.hip for what it computes).
//
// 16-bit rows: a workgroup takes 128 columns of one K/V head of one sequence, a column being a (new token, query head that reads this K/V head),
// heads fastest: with G query heads to a K/V head a row of the pool is read once for G heads of 128 / G tokens. It walks the
// tokens that these see in tiles of 64, or a share of them. Its four waves own 32 columns each.
//   * S^T = K . Q^T (32x32x16): a lane holds 16 scores of ONE column, so the running maximum and sum of the softmax are the lane's and one
//     lane swap away, and its probabilities, rounded once to the rows' type, are as they lie the operand P^T of O^T += V^T . P^T.
//     Rounding a probability costs half a step of the type relative to it, about what the rounding of the result costs; two parts
//     would take half as many matrix instructions again. fp16 probabilities are taken times 2^7, so that they keep all their bits
//     down to 2^-21 of the largest. The sum below the fraction line is that of the rounded ones (a row of ones on the pipe).
//   * K and V rows go from the pool straight into a two-stage LDS ring (global_load_lds, an address per 16 bytes): slots are read a
//     tile ahead of the copy, a lane each, and handed round. Pieces are XOR-swizzled on the way; V is read through the transposing LDS read.
//   * one barrier per tile, between its softmax and its P.V; K of tile t + 2 and V of t + 1 are asked for right behind it.
//   * the running maximum is replaced only when a score exceeds it by more than 2^8.
//   * a workgroup finds its piece of work in the lengths on the device: the grid is as large as the rows of q can make it, and sequences
//     of one new token and of thousands are dealt alike. The pieces of one K/V head's sequence are neighbours on one XCD.
//   * shares of a sequence leave (maximum, sum, weighted sum of V) in workspace, which pagedMergeKernel joins.
// What a column does not see (later tokens, those before the window, slots outside the pool) has no score; but a weight of zero does not
// keep an infinity or NaN in V out of a sum, and scores beyond 2^22 would be off against their rounded maximum. A column whose sums come
// out not finite, or whose maximum is beyond that, is walked again by itself on the vector ALUs, the tokens that it sees alone (PaColumn).
#include <algorithm>
#include <type_traits>

#include "paged_attention.hpp"

namespace amd {

constexpr int kPtCols = 128, kPtTile = 64;
constexpr float kPtRescaleStep = 8.0f;            // log2 domain
constexpr float kPtLargeScore = 4194304.f;        // 2^22: a maximum beyond it has no more than two places below one
constexpr int kPtMaxSplit = 64;                   // pagedMergeKernel has a lane for each

template <typename T>
struct PtMfma;
template <>
struct PtMfma<bf16_t> {
  typedef bf16x8 Frag;
  typedef bf16x4 Half;
  static constexpr float kRaise = 0.f;  // log2 of what probabilities are multiplied by
  static __device__ __forceinline__ f32x16 run(Frag a, Frag b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
};
template <>
struct PtMfma<half_t> {
  typedef f16x8 Frag;
  typedef f16x4 Half;
  static constexpr float kRaise = 7.f;
  static __device__ __forceinline__ f32x16 run(Frag a, Frag b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
};

struct PtArgs {
  PaArgs a;
  float* partial;    // [rows, heads, splits, 2 + d]
  int splits, tilesPerSplit;
  unsigned kSlotBytes, vSlotBytes;
};

// The tiles that the tokens at positions pMin ... pMax see: sinkTiles of the sequence's first tokens, the others from token `low` on, up
// to pMax. Without a gap between the two, from token 0 on.
struct PtSpan {
  int low, end, sinks, sinkTiles, tiles;
  __device__ __forceinline__ PtSpan(const PaArgs& a, int pMin, int pMax) {
    end = pMax + 1, sinks = a.sinks;
    low = max(0, pMin - a.window + 1);
    sinkTiles = (min(sinks, low) + kPtTile - 1) / kPtTile;
    if (low <= sinkTiles * kPtTile) sinkTiles = 0, low = 0;
    tiles = end <= 0 ? 0 : sinkTiles + (end - low + kPtTile - 1) / kPtTile;
  }
  __device__ __forceinline__ int base(int tile) const { return tile < sinkTiles ? tile * kPtTile : low + (tile - sinkTiles) * kPtTile; }
  __device__ __forceinline__ int limit(int tile) const { return tile < sinkTiles ? sinks : end; }
};

// Blocks of columns of a sequence, and the most shares that one of them has.
template <int COLS>
struct PtPieces {
  int blocks, splits;
  __device__ __forceinline__ PtPieces(const PtArgs& x, const PaSequence& s) {
    const int group = x.a.heads / x.a.kvHeads, tokens = s.end - s.first;
    blocks = (int)(((int64_t)tokens * group + COLS - 1) / COLS);
    const int upTo = (s.origin + s.end + kPtTile - 1) / kPtTile;
    const int64_t windowed = (x.a.sinks + kPtTile - 1) / kPtTile + ((int64_t)x.a.window + kPtCols + kPtTile - 1) / kPtTile;
    splits = max(1, ((int)min((int64_t)upTo, windowed) + x.tilesPerSplit - 1) / x.tilesPerSplit);
  }
  __device__ __forceinline__ int all() const { return blocks * splits; }
};

// XOR on the 16-byte piece index of a row in LDS: K so that 32 rows' pieces of one index, V so that the row pieces of a transposing read
// fall on different banks.
template <int D>
__device__ __forceinline__ int ptSwizzleK(int key) { return D >= 128 ? (key & 15) : ((key >> 1) & 7); }
template <int D>
__device__ __forceinline__ int ptSwizzleV(int key) { return D >= 128 ? 4 * (key & 3) : 4 * ((key >> 1) & 1); }

// Column `col` of a piece of work by itself, on the vector ALUs of one wave.
template <typename T, int D>
__device__ __forceinline__ void pagedAgain(const PtArgs& x, const PaSequence& s, int kvh, int64_t locBase, const PtSpan& span, int t0, int t1, int split, bool whole,
                                           int col) {
  const PaArgs& a = x.a;
  const int lane = threadIdx.x & 63, group = a.heads / a.kvHeads, token = s.first + col / group, h = kvh * group + col % group, p = s.origin + token;
  const int64_t row = s.start + token;
  int head, low;
  paSeen(a, p, &head, &low);
  // of the tiles' tokens those that it sees: of the first ones, and of the others
  const int from = span.base(max(t0, span.sinkTiles)), to = t1 > span.sinkTiles ? min(span.base(t1), p + 1) : 0;
  const int first0 = span.sinkTiles > 0 ? min(t0, span.sinkTiles) * kPtTile : from, first1 = span.sinkTiles > 0 ? min(head, min(t1, span.sinkTiles) * kPtTile) : min(head, to);
  PaColumn<T, D / 64, (D > 128 ? 4 : 8)> one;
  one.walk(a, reinterpret_cast<const T*>(a.q) + row * a.qTok + (int64_t)h * a.qHead, kvh, locBase, first0, first1, max(from, low), to, 0, 64);
  float* dst = x.partial + ((row * a.heads + h) * x.splits + split) * (2 + a.d);
  T* out = reinterpret_cast<T*>(a.out) + row * a.oTok + (int64_t)h * a.oHead;
  const float inv = one.l == 0.f ? 0.f : 1.f / one.l;
  if (!whole && lane == 0) dst[0] = one.m, dst[1] = one.l;
#pragma unroll
  for (int j = 0; j < D / 64; ++j) {
    const int e = lane + 64 * j;
    if (e >= a.d) continue;
    if (whole) out[e] = static_cast<T>(one.acc[j] * inv);
    else dst[2 + e] = one.acc[j];
  }
}

// One block of columns over tiles [t0, t1), all of them if `whole`.
// D: the head size that tiles are laid out for; with PART a.d is any multiple of 8 below it, and the places behind it are zeros.
template <typename T, int D, bool PART>
__device__ __forceinline__ void pagedTileBlock(const PtArgs& x, const PaSequence& s, int b, int kvh, int block, const PtSpan& span, int t0, int t1, int split,
                                               bool whole) {
  using M = PtMfma<T>;
  using Frag = typename M::Frag;
  using Half = typename M::Half;
  constexpr int KS = D / 16, DT = D / 32, CPR = D / 8, RPL = 64 / CPR, NLD = kPtTile / RPL / 4, STAGE = kPtTile * D;
  constexpr int ROWB = D * (int)sizeof(T);
  constexpr unsigned kStageBytes = STAGE * sizeof(T);
  extern __shared__ __attribute__((aligned(16))) char ptSmem[];
  const PaArgs& a = x.a;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l31 = lane & 31, half = lane >> 5;
  const int group = a.heads / a.kvHeads, cols = (s.end - s.first) * group, c0 = block * kPtCols + wave * 32;
  const bool waveLives = c0 < cols;
  const int col = min(c0 + l31, cols - 1), token = s.first + col / group, h = kvh * group + col % group;
  const int p = s.origin + token;
  const int64_t row = s.start + token;
  const int pFirst = __builtin_amdgcn_readlane(p, 0), pLast = __builtin_amdgcn_readlane(p, 31);
  const int window = a.window, sinksSeen = max(0, min(a.sinks, p + 1));
  const int64_t locBase = (int64_t)b * a.locRowStride + (a.maxLen - s.len);

  Frag qf[KS];
  {
    const T* q = reinterpret_cast<const T*>(a.q) + row * a.qTok + (int64_t)h * a.qHead;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      if (!PART || ks * 16 + half * 8 < a.d) {
        qf[ks] = *reinterpret_cast<const Frag*>(q + ks * 16 + half * 8);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) qf[ks][e] = static_cast<T>(0.f);
      }
    }
  }

  // ---- slots: lane l has that of token l of a tile; past the tile's last token that again (whose place has no score)
  auto askSlot = [&](int t) {
    if (t >= t1) return (int64_t)0;
    return ldIndex(a.bLoc, locBase + min(span.base(t) + lane, span.limit(t) - 1), a.loc64);
  };
  auto inPool = [&](int64_t slot) { return slot >= 0 && slot < a.slots; };
  // ---- tile copies. Copy instruction i of this wave fills the 1 KiB (i * 4 + wave) of a stage: lane l the place (row l / CPR, piece l % CPR),
  // for which it fetches the piece that the swizzle puts there.
  int kPiece[NLD], vPiece[NLD];
#pragma unroll
  for (int i = 0; i < NLD; ++i) {
    const int key = (i * 4 + wave) * RPL + lane / CPR, pc = lane % CPR;
    kPiece[i] = (pc ^ ptSwizzleK<D>(key)) << 4, vPiece[i] = (pc ^ ptSwizzleV<D>(key)) << 4;  // bytes
  }
  const char* const kBase = reinterpret_cast<const char*>(reinterpret_cast<const T*>(a.k) + kvh * a.kHeadStride);
  const char* const vBase = reinterpret_cast<const char*>(reinterpret_cast<const T*>(a.v) + kvh * a.vHeadStride);
  const unsigned ldsK0 = (unsigned)(uintptr_t)ptSmem, ldsV0 = ldsK0 + 2 * kStageBytes;
  // (slots outside the pool are skipped, never dereferenced: the tile's first one inside stands in, slot 0 where there is none)
  auto rowsOf = [&](int64_t slot, uint64_t in, int (&rows)[NLD]) {
    const int instead = in != 0 ? __builtin_amdgcn_readlane((int)slot, __builtin_ctzll(in)) : 0;
    const int mine = inPool(slot) ? (int)slot : instead;
#pragma unroll
    for (int i = 0; i < NLD; ++i) rows[i] = __shfl(mine, (i * 4 + wave) * RPL + lane / CPR, 64);
  };
  auto copyTile = [&](const char* base, const int (&rows)[NLD], unsigned slotBytes, const int (&piece)[NLD], unsigned to) {
#pragma unroll
    for (int i = 0; i < NLD; ++i) {
      const char* from = base + ((uint64_t)(unsigned)rows[i] * slotBytes + (unsigned)piece[i]);
      if (!PART || piece[i] < a.d * (int)sizeof(T)) globalLoadToLds16(from, to + (unsigned)wave * 1024u + i * 4096u);
    }
  };
  auto copyK = [&](const int (&rows)[NLD], int stage) { copyTile(kBase, rows, x.kSlotBytes, kPiece, ldsK0 + stage * kStageBytes); };
  auto copyV = [&](const int (&rows)[NLD], int stage) { copyTile(vBase, rows, x.vSlotBytes, vPiece, ldsV0 + stage * kStageBytes); };

  f32x16 o[DT];
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
#pragma unroll
    for (int r = 0; r < 16; ++r) o[dt][r] = 0.f;
  float m = -INFINITY, l = 0.f;  // m: in units of log2
  const float scale2 = a.scaleLog2e;

  auto tileBarrier = []() {  // what this wave has in flight is done, then the workgroup meets
    __builtin_amdgcn_s_waitcnt(0x0070);
    __builtin_amdgcn_s_barrier();
  };
  constexpr int NS = 2 * KS, kKAhead = 4;
  Frag kfr[kKAhead + 1];
  const int kswz = ptSwizzleK<D>(l31);
  const unsigned kLane = (unsigned)(l31 * ROWB + ((half ^ (kswz & 1)) << 4) + ((kswz >> 1) << 5));
  typedef __attribute__((address_space(3))) const Frag* LdsFrag;
  auto kfragAt = [&](unsigned at, int i) {
    return *(LdsFrag)(uintptr_t)((at ^ (unsigned)((i >> 1) << 5)) + (unsigned)((i & 1) * 32 * ROWB));
  };
  auto opaque = [](unsigned v) {
    asm volatile("" : "+v"(v));
    return v;
  };

  if (PART) {  // the places behind a row's end stay zeros: no copy fills them
    for (unsigned i = tid * 16; i < 4 * kStageBytes; i += 256 * 16) *reinterpret_cast<u32x4*>(ptSmem + i) = u32x4{0, 0, 0, 0};
    __syncthreads();
  }
  int rowsNext[NLD], rowsAfter[NLD];      // of tiles t + 1 and t + 2
  uint64_t valid, validNext, validAfter;  // tokens of tiles t, t + 1, t + 2 whose slot is in the pool
  int64_t asked;                          // slots of tile t + 3
  {
    const int64_t first = askSlot(t0), second = askSlot(t0 + 1), third = askSlot(t0 + 2);
    int rows[NLD];
    valid = __builtin_amdgcn_ballot_w64(inPool(first));
    validNext = __builtin_amdgcn_ballot_w64(inPool(second)), validAfter = __builtin_amdgcn_ballot_w64(inPool(third));
    rowsOf(first, valid, rows);
    if (t0 < t1) {
      copyK(rows, 0);
      copyV(rows, 0);
    }
    rowsOf(second, validNext, rowsNext), rowsOf(third, validAfter, rowsAfter);
  }
  tileBarrier();
  if (t0 + 1 < t1) copyK(rowsNext, 1);
  asked = askSlot(t0 + 3);
#pragma unroll
  for (int i = 0; i < kKAhead; ++i) kfr[i] = kfragAt(kLane + ldsK0, i);

  for (int t = t0; t < t1; ++t) {
    const int cur = (t - t0) & 1, k0 = span.base(t);
    // wave-uniform: whether a column sees any of the tile, and whether all see all of it
    const bool live = waveLives && k0 <= pLast && (k0 + kPtTile - 1 > pFirst - window || k0 < a.sinks);
    const bool all = k0 + kPtTile - 1 <= pFirst && (k0 > pLast - window || k0 + kPtTile <= a.sinks) && valid == ~0ull;
    const unsigned kCur = opaque(kLane + ldsK0 + cur * kStageBytes), kOther = opaque(kLane + ldsK0 + (cur ^ 1) * kStageBytes);
    f32x16 sc[2];
    if (live) {
#pragma unroll
      for (int kt2 = 0; kt2 < 2; ++kt2)
#pragma unroll
        for (int r = 0; r < 16; ++r) sc[kt2][r] = 0.f;
      __builtin_amdgcn_s_setprio(1);  // (a wave in its products goes before one in its softmax)
#pragma unroll
      for (int i = 0; i < NS; ++i) {
        if (i + kKAhead < NS) kfr[(i + kKAhead) % (kKAhead + 1)] = kfragAt(kCur, i + kKAhead);
        sc[i & 1] = M::run(kfr[i % (kKAhead + 1)], qf[i >> 1], sc[i & 1]);
        __builtin_amdgcn_sched_barrier(0);
      }
      __builtin_amdgcn_s_setprio(0);
      if (!all) {
#pragma unroll
        for (int kt2 = 0; kt2 < 2; ++kt2)
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            const int bit = (r >> 2) * 8 + (r & 3), kj = k0 + kt2 * 32 + half * 4 + bit;
            const uint32_t in = (uint32_t)(valid >> (kt2 * 32)) >> (half * 4);
            if (!((unsigned)(p - kj) < (unsigned)window || kj < sinksSeen) || (in >> bit & 1) == 0) sc[kt2][r] = -INFINITY;
          }
      }
      float mt = -INFINITY;
#pragma unroll
      for (int kt2 = 0; kt2 < 2; ++kt2)
#pragma unroll
        for (int r = 0; r < 16; ++r) mt = fmaxf(mt, sc[kt2][r]);
      {  // the other half of the wave holds the other scores of the column
        const auto sw = __builtin_amdgcn_permlane32_swap(__float_as_uint(mt), __float_as_uint(mt), false, false);
        mt = fmaxf(__uint_as_float(sw[0]), __uint_as_float(sw[1])) * scale2;
      }
      // (nothing seen so far: mn stays minus infinity, and scores are taken against 0)
      const float mn = mt - m > kPtRescaleStep ? mt : m;
      const float ref = mn == -INFINITY ? 0.f : mn;
      const float raised = ref - M::kRaise;
#pragma unroll
      for (int kt2 = 0; kt2 < 2; ++kt2)
#pragma unroll
        for (int r = 0; r < 16; ++r)
          sc[kt2][r] = __builtin_amdgcn_exp2f(fmaf(sc[kt2][r], scale2, -raised));
      if (__builtin_amdgcn_ballot_w64(mn > m) != 0) {
        const float corr = __builtin_amdgcn_exp2f(m - ref);
        l *= corr;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
          for (int r = 0; r < 16; ++r) o[dt][r] *= corr;
        m = mn;
      }
    }
    tileBarrier();
    if (t + 2 < t1) copyK(rowsAfter, cur);
    if (t + 1 < t1) copyV(rowsNext, cur ^ 1);
    if (live) {
      __builtin_amdgcn_s_setprio(2);
      constexpr int NPV = 4 * DT, kVAhead = 3;
      const int trKey = half * 4 + ((lane & 15) >> 2);
      const int trChunk = ((lane >> 4) & 1) * 2 + ((lane & 3) >> 1), trIn = (lane & 1) * 4;
      const int vsw = D >= 128 ? (trKey & 3) : ((trKey >> 1) & 1);
      const unsigned vCur = opaque((unsigned)(trKey * ROWB + (trChunk << 4) + trIn * 2 + (vsw << 6)) + ldsV0 + cur * kStageBytes);
      typedef __attribute__((address_space(3))) s16x4* LdsTr;
      auto vfrag = [&](int i) {
        const int g = i / DT, dt = i % DT;  // key group of 16, d tile
        Half part[2];
#pragma unroll
        for (int r = 0; r < 2; ++r)
          part[r] = __builtin_bit_cast(Half, __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsTr)(uintptr_t)((vCur ^ (unsigned)(dt << 6)) + (unsigned)((g * 16 + r * 8) * ROWB))));
        Frag vf;
        vf[0] = part[0][0], vf[1] = part[0][1], vf[2] = part[0][2], vf[3] = part[0][3];
        vf[4] = part[1][0], vf[5] = part[1][1], vf[6] = part[1][2], vf[7] = part[1][3];
        return vf;
      };
      Frag vfr[kVAhead + 1];
#pragma unroll
      for (int i = 0; i < kVAhead; ++i) vfr[i] = vfrag(i);
      Frag pf, ones;
#pragma unroll
      for (int j = 0; j < 8; ++j) ones[j] = static_cast<T>(1.0f);
      f32x16 lsum;
#pragma unroll
      for (int r = 0; r < 16; ++r) lsum[r] = 0.f;
#pragma unroll
      for (int i = 0; i < NPV; ++i) {
        const int g = i / DT, dt = i % DT;
        if (dt == 0) {
#pragma unroll
          for (int j = 0; j < 8; ++j) pf[j] = static_cast<T>(sc[g >> 1][8 * (g & 1) + j]);
          lsum = M::run(ones, pf, lsum);
        }
        if (i + kVAhead < NPV) vfr[(i + kVAhead) % (kVAhead + 1)] = vfrag(i + kVAhead);
        if (i >= NPV - kKAhead) kfr[i - (NPV - kKAhead)] = kfragAt(kOther, i - (NPV - kKAhead));  // the next tile's first K fragments
        o[dt] = M::run(vfr[i % (kVAhead + 1)], pf, o[dt]);
        __builtin_amdgcn_sched_barrier(0);
      }
      l += lsum[0];
      __builtin_amdgcn_s_setprio(0);
    } else {
#pragma unroll
      for (int i = 0; i < kKAhead; ++i) kfr[i] = kfragAt(kOther, i);
    }
    // (behind the copies: their wait is the next barrier's, and so is this one's)
    valid = validNext, validNext = validAfter;
#pragma unroll
    for (int i = 0; i < NLD; ++i) rowsNext[i] = rowsAfter[i];
    validAfter = __builtin_amdgcn_ballot_w64(inPool(asked));
    rowsOf(asked, validAfter, rowsAfter);
    asked = askSlot(t + 4);
  }

  // ---- columns that have to be walked again, as bits (those past the last one are copies of it)
  uint32_t again;
  {
    uint32_t largest = __float_as_uint(l) & 0x7fffffffu;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int r = 0; r < 16; ++r) largest = max(largest, __float_as_uint(o[dt][r]) & 0x7fffffffu);
    const uint64_t bad = __builtin_amdgcn_ballot_w64(c0 + l31 < cols && (largest >= 0x7f800000u || (m != -INFINITY && !(fabsf(m) < kPtLargeScore))));
    again = (uint32_t)bad | (uint32_t)(bad >> 32);
  }
  __syncthreads();  // (the output takes the place of the stages)
  if (!whole) {
    if (c0 + l31 < cols && (again >> l31 & 1) == 0) {
      float* dst = x.partial + ((row * a.heads + h) * x.splits + split) * (2 + a.d);
      if (half == 0) dst[0] = m - M::kRaise, dst[1] = l;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const int e = dt * 32 + g * 8 + half * 4;
          if (PART && e >= a.d) continue;
          *reinterpret_cast<float2*>(dst + 2 + e) = float2{o[dt][g * 4], o[dt][g * 4 + 1]};
          *reinterpret_cast<float2*>(dst + 4 + e) = float2{o[dt][g * 4 + 2], o[dt][g * 4 + 3]};
        }
    }
  } else {
    // O^T (lane = column) -> LDS [column][d] -> 16-byte stores
    constexpr int OS = D + 8;  // padded row, elements
    T* sO = reinterpret_cast<T*>(ptSmem) + wave * 32 * OS;
    const float inv = l > 0.f ? 1.f / l : 0.f;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        Half part;
#pragma unroll
        for (int e = 0; e < 4; ++e) part[e] = static_cast<T>(o[dt][g * 4 + e] * inv);
        *reinterpret_cast<Half*>(sO + l31 * OS + dt * 32 + g * 8 + half * 4) = part;
      }
    exchangeInWave();
#pragma unroll
    for (int i = 0; i < 32 * CPR / 64; ++i) {
      const int chunk = lane + 64 * i, r = chunk / CPR, c = chunk % CPR;
      const int oc = c0 + r, tok = s.first + oc / group;
      if (oc < cols && (again >> r & 1) == 0 && (!PART || c * 8 < a.d))
        *reinterpret_cast<Frag*>(reinterpret_cast<T*>(a.out) + (s.start + tok) * a.oTok + (int64_t)(kvh * group + oc % group) * a.oHead + c * 8) =
            *reinterpret_cast<const Frag*>(sO + r * OS + c * 8);
  }
  }
  for (; again != 0; again &= again - 1) pagedAgain<T, D>(x, s, kvh, locBase, span, t0, t1, split, whole, c0 + __builtin_ctz(again));
}

// A workgroup's pieces of work. grid: K/V heads fastest (the ids go round the XCDs, so a head's pieces stay on one), then the list of
// pieces: sequence after sequence, shares from the first, blocks from the last, which has the most tiles.
template <int COLS, typename F>
__device__ __forceinline__ void pagedPieces(const PtArgs& x, F&& walk) {
  const PaArgs& a = x.a;
  const int kvh = blockIdx.x % a.kvHeads, step = gridDim.x / a.kvHeads, group = a.heads / a.kvHeads;
  for (int64_t u = blockIdx.x / a.kvHeads;; u += step) {
    const PaPlace at = paFind(a, u, [&](const PaSequence& s) { return PtPieces<COLS>(x, s).all(); });
    if (at.b < 0) return;
    const PaSequence& s = at.s;
    const PtPieces<COLS> pieces(x, s);
    const int split = at.at / pieces.blocks, block = pieces.blocks - 1 - at.at % pieces.blocks;
    const int cols = (s.end - s.first) * group, origin = s.origin + s.first;
    const PtSpan span(a, origin + block * COLS / group, origin + min(block * COLS + COLS - 1, cols - 1) / group);
    const bool whole = span.tiles <= x.tilesPerSplit;
    const int t0 = split * x.tilesPerSplit, t1 = min(span.tiles, t0 + x.tilesPerSplit);
    if (split == 0 || t0 < span.tiles) walk(s, at.b, kvh, block, span, t0, t1, split, whole);
    if (u + step >= at.total) return;
    __syncthreads();  // (the next piece's tiles take the place of this one's output)
  }
}

template <typename T, int D, bool PART>
__global__ __launch_bounds__(256, D > 128 ? 1 : 2) void pagedTileKernel(PtArgs x) {
  pagedPieces<kPtCols>(x, [&](const PaSequence& s, int b, int kvh, int block, const PtSpan& span, int t0, int t1, int split, bool whole) {
    pagedTileBlock<T, D, PART>(x, s, b, kvh, block, span, t0, t1, split, whole);
  });
}

// fp32 rows on the fp32 matrix instructions (true fp32 products and sums). A workgroup takes 16 columns; of every tile its four waves take 16
// tokens each, with a softmax state of their own, and the states meet in LDS at the end: the chains of loads are short, which is what bounds
// the short sequences of the fp32 configuration.
// v_mfma_f32_16x16x4_f32: lane (c = l & 15, g = l >> 4) feeds row c, k = g of both operands and receives D[4 g + r][c].
//   S^T = K Q^T: the contraction order is free as long as both operands agree, so group g takes the D / 4 consecutive elements from g D / 4
//   on, 16-byte loads straight into operand registers. The lane ends up with tokens 4 g .. 4 g + 3 of column c, which is P^T's operand
//   layout when step r takes token 4 g + r from group g: no data moves between lanes.
//   O^T = V^T P^T: row i of output tile t stands for element i (D / 16) + t, so a lane's D / 16 operands of a token are consecutive in memory,
//   and its results are D / 4 consecutive elements of column c.
// Rows go from the pool into registers a tile ahead, slots another one.
constexpr int kPtFloatCols = 16;
template <int D, bool PART>
__device__ __forceinline__ void pagedFloatBlock(const PtArgs& x, const PaSequence& s, int b, int kvh, int block, const PtSpan& span, int t0, int t1, int split,
                                                bool whole) {
  constexpr int S = D / 4, E = D / 16, PITCH = D + 4;
  extern __shared__ __attribute__((aligned(16))) char ptSmem[];
  float* const so = reinterpret_cast<float*>(ptSmem);  // [4][16][PITCH]
  __shared__ float sm[4][16], sl[4][16];
  const PaArgs& a = x.a;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), c = lane & 15, g = lane >> 4;
  const int group = a.heads / a.kvHeads, cols = (s.end - s.first) * group, c0 = block * kPtFloatCols;
  const int col = min(c0 + c, cols - 1), token = s.first + col / group, h = kvh * group + col % group, p = s.origin + token;
  const int pFirst = __builtin_amdgcn_readlane(p, 0), pLast = __builtin_amdgcn_readlane(p, 15);
  const int window = a.window, sinksSeen = max(0, min(a.sinks, p + 1));
  const int64_t locBase = (int64_t)b * a.locRowStride + (a.maxLen - s.len);
  const float* const kHead = reinterpret_cast<const float*>(a.k) + kvh * a.kHeadStride;
  const float* const vHead = reinterpret_cast<const float*>(a.v) + kvh * a.vHeadStride;
  f32x4 qf[S / 4], kf[2][S / 4], vf[2][4][E / 4], o[E];
  // (PART: places past the row's end read its first piece, are zeros in q and K, and give elements that are not stored)
  auto at = [&](int e) { return !PART || e < a.d ? e : 0; };
  {
    const float* q = reinterpret_cast<const float*>(a.q) + (s.start + token) * a.qTok + (int64_t)h * a.qHead;
#pragma unroll
    for (int i = 0; i < S / 4; ++i) {
      qf[i] = *reinterpret_cast<const f32x4*>(q + at(g * S + 4 * i));
      if (PART && g * S + 4 * i >= a.d) qf[i] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
  }
  auto askSlot = [&](int t) {
    if (t >= t1) return (int64_t)0;
    return ldIndex(a.bLoc, locBase + min(span.base(t) + 16 * wave + c, span.limit(t) - 1), a.loc64);
  };
  uint32_t valid[2];
  auto fetch = [&](int64_t slot, auto buf) {
    constexpr int B = decltype(buf)::value;
    const bool in = slot >= 0 && slot < a.slots;
    valid[B] = (uint32_t)__builtin_amdgcn_ballot_w64(in) & 0xffffu;
    // (slots outside the pool are skipped, never dereferenced: the first one inside stands in, slot 0 where there is none)
    const int instead = valid[B] != 0 ? __builtin_amdgcn_readlane((int)slot, __builtin_ctz(valid[B])) : 0, mine = in ? (int)slot : instead;
    const float* kr = kHead + (int64_t)mine * a.kSlotStride;
#pragma unroll
    for (int i = 0; i < S / 4; ++i) {
      kf[B][i] = *reinterpret_cast<const f32x4*>(kr + at(g * S + 4 * i));
      if (PART && g * S + 4 * i >= a.d) kf[B][i] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const float* vr = vHead + (int64_t)__shfl(mine, 4 * g + r, 64) * a.vSlotStride;
#pragma unroll
      for (int i = 0; i < E / 4; ++i) vf[B][r][i] = *reinterpret_cast<const f32x4*>(vr + at(c * E + 4 * i));
    }
  };
#pragma unroll
  for (int i = 0; i < E; ++i) o[i] = f32x4{0.f, 0.f, 0.f, 0.f};
  float m = -INFINITY, l = 0.f;  // m: in units of log2
  auto tile = [&](int t, auto buf) {
    constexpr int B = decltype(buf)::value;
    const int k0 = span.base(t) + 16 * wave;
    if (k0 > pLast || k0 >= span.limit(t) || (k0 + 15 <= pFirst - window && k0 >= a.sinks)) return;  // (uniform: nobody sees any of it)
    f32x4 acc[2] = {f32x4{0.f, 0.f, 0.f, 0.f}, f32x4{0.f, 0.f, 0.f, 0.f}};  // two chains: half the dependent latency
#pragma unroll
    for (int i = 0; i < S; ++i) acc[i & 1] = __builtin_amdgcn_mfma_f32_16x16x4f32(kf[B][i >> 2][i & 3], qf[i >> 2][i & 3], acc[i & 1], 0, 0, 0);
    float w[4], mx = m;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int kj = k0 + 4 * g + r;
      const bool sees = ((unsigned)(p - kj) < (unsigned)window || kj < sinksSeen) && (valid[B] >> (4 * g + r) & 1) != 0;
      w[r] = sees ? (acc[0][r] + acc[1][r]) * a.scaleLog2e : -INFINITY;
      mx = fmaxf(mx, w[r]);
    }
    mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
    mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
    const float ref = mx == -INFINITY ? 0.f : mx, keep = exp2f(m - ref);
    m = mx, l *= keep;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      w[r] = exp2f(behindRounded(w[r], ref));
      l += w[r];
    }
#pragma unroll
    for (int i = 0; i < E; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) o[i][r] *= keep;
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int i = 0; i < E; ++i) o[i] = __builtin_amdgcn_mfma_f32_16x16x4f32(vf[B][r][i >> 2][i & 3], w[r], o[i], 0, 0, 0);
  };
  using B0 = std::integral_constant<int, 0>;
  using B1 = std::integral_constant<int, 1>;
  if (t0 < t1) {
    const int64_t first = askSlot(t0);
    int64_t next = askSlot(t0 + 1);
    fetch(first, B0{});
    for (int t = t0; t < t1; t += 2) {
      if (t + 1 < t1) {
        const int64_t slot = next;
        next = askSlot(t + 2);
        fetch(slot, B1{});
      }
      tile(t, B0{});
      if (t + 1 >= t1) break;
      if (t + 2 < t1) {
        const int64_t slot = next;
        next = askSlot(t + 3);
        fetch(slot, B0{});
      }
      tile(t + 1, B1{});
    }
  }
  l += __shfl_xor(l, 16, 64);
  l += __shfl_xor(l, 32, 64);
  if (l != l && m == -INFINITY) m = 0.f;  // scores that are not numbers alone: as a maximum of minus infinity they would be left out
  if (g == 0) sm[wave][c] = m, sl[wave][c] = l;
#pragma unroll
  for (int r = 0; r < 4; ++r)
#pragma unroll
    for (int i = 0; i < E / 4; ++i)
      *reinterpret_cast<f32x4*>(so + (wave * 16 + c) * PITCH + (4 * g + r) * E + 4 * i) = f32x4{o[4 * i][r], o[4 * i + 1][r], o[4 * i + 2][r], o[4 * i + 3][r]};
  __syncthreads();
  // a column to 16 lanes
  const int mine = threadIdx.x >> 4, e0 = c * E, oc = c0 + mine, at0 = s.first + min(oc, cols - 1) / group, hc = kvh * group + min(oc, cols - 1) % group;
  const int64_t row = s.start + at0;
  float mAll = -INFINITY, sum = 0.f;
#pragma unroll
  for (int w = 0; w < 4; ++w) mAll = fmaxf(mAll, sm[w][mine]);
  f32x4 v[E / 4] = {};
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    const float weight = sm[w][mine] == -INFINITY ? 0.f : exp2f(sm[w][mine] - mAll);
    sum += sl[w][mine] * weight;
#pragma unroll
    for (int i = 0; i < E / 4; ++i)
#pragma unroll
      for (int k = 0; k < 4; ++k) v[i][k] += so[(w * 16 + mine) * PITCH + e0 + 4 * i + k] * weight;
  }
  bool odd = !(fabsf(sum) < INFINITY);
#pragma unroll
  for (int i = 0; i < E / 4; ++i)
#pragma unroll
    for (int k = 0; k < 4; ++k) odd |= !(fabsf(v[i][k]) < INFINITY);
  // columns whose sums are not finite: by themselves, with the tokens that they see alone
  const uint64_t bad = __builtin_amdgcn_ballot_w64(odd && oc < cols);
  const bool again = (bad >> (lane & 48) & 0xffffu) != 0;
  if (oc < cols && !again) {
    if (whole) {
      const float inv = sum == 0.f ? 0.f : 1.f / sum;
      float* out = reinterpret_cast<float*>(a.out) + row * a.oTok + (int64_t)hc * a.oHead + e0;
#pragma unroll
      for (int i = 0; i < E / 4; ++i)
        if (!PART || e0 + 4 * i < a.d) *reinterpret_cast<f32x4*>(out + 4 * i) = v[i] * inv;
    } else {
      float* dst = x.partial + ((row * a.heads + hc) * x.splits + split) * (2 + a.d);
      if (c == 0) dst[0] = mAll, dst[1] = sum;
#pragma unroll
      for (int i = 0; i < E / 4; ++i) {
        if (PART && e0 + 4 * i >= a.d) continue;
        *reinterpret_cast<float2*>(dst + 2 + e0 + 4 * i) = float2{v[i][0], v[i][1]};
        *reinterpret_cast<float2*>(dst + 4 + e0 + 4 * i) = float2{v[i][2], v[i][3]};
      }
    }
  }
  for (int i = 0; i < 4; ++i)
    if ((bad >> (16 * i) & 0xffffu) != 0) pagedAgain<float, D>(x, s, kvh, locBase, span, t0, t1, split, whole, c0 + 4 * wave + i);
}

template <int D, bool PART>
__global__ __launch_bounds__(256) void pagedFloatKernel(PtArgs x) {
  pagedPieces<kPtFloatCols>(x, [&](const PaSequence& s, int b, int kvh, int block, const PtSpan& span, int t0, int t1, int split, bool whole) {
    pagedFloatBlock<D, PART>(x, s, b, kvh, block, span, t0, t1, split, whole);
  });
}

// out of the rows whose block was walked in shares: a wave per (row, head). Lane i takes maximum and sum of share i, then every lane its
// elements of all of them.
template <typename T, int COLS>
__global__ __launch_bounds__(256) void pagedMergeKernel(PtArgs x) {
  constexpr int kPerLane = 4, kBatch = 8;  // d <= 256; shares whose elements are asked for at once
  const PaArgs& a = x.a;
  const int lane = threadIdx.x & 63, group = a.heads / a.kvHeads;
  const int64_t step = (int64_t)gridDim.x * 4;
  for (int64_t pair = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);; pair += step) {
    const PaPlace at = paFind(a, pair / a.heads, [](const PaSequence& s) { return s.end - s.first; });
    if (at.b < 0) return;
    const PaSequence& s = at.s;
    const int h = (int)(pair % a.heads), cols = (s.end - s.first) * group, origin = s.origin + s.first;
    const int block = (at.at * group + h % group) / COLS;
    const PtSpan span(a, origin + block * COLS / group, origin + min(block * COLS + COLS - 1, cols - 1) / group);
    const int shares = (span.tiles + x.tilesPerSplit - 1) / x.tilesPerSplit;
    if (shares > 1) {
      const int64_t row = s.start + s.first + at.at;
      const float* src = x.partial + (row * a.heads + h) * x.splits * (2 + a.d);
      const int mine = min(lane, shares - 1);
      float m = src[mine * (2 + a.d)], l = src[mine * (2 + a.d) + 1], acc[kPerLane] = {0.f, 0.f, 0.f, 0.f};
      if (lane >= shares) m = -INFINITY, l = 0.f;
      const float most = waveMax(m);
      float w = m == -INFINITY ? 0.f : exp2f(m - most);
      if (l != l) w = l;  // (scores that are not numbers alone have no maximum)
      const uint64_t none = __builtin_amdgcn_ballot_w64(w == 0.f && m == -INFINITY);  // shares without a score
      const float sum = waveSum(l * w);
      for (int i0 = 0; i0 < shares; i0 += kBatch) {
        float v[kBatch][kPerLane];
#pragma unroll
        for (int i = 0; i < kBatch; ++i)
#pragma unroll
          for (int k = 0; k < kPerLane; ++k) {
            const int e = lane + 64 * k;
            v[i][k] = e < a.d ? src[min(i0 + i, shares - 1) * (2 + a.d) + 2 + e] : 0.f;
          }
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
          if (i0 + i >= shares) break;
          const float wi = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, w), i0 + i));
          if (none >> (i0 + i) & 1) continue;
#pragma unroll
          for (int k = 0; k < kPerLane; ++k) acc[k] += wi * v[i][k];
        }
      }
      const float inv = sum == 0.f ? 0.f : 1.f / sum;
      T* out = reinterpret_cast<T*>(a.out) + row * a.oTok + h * a.oHead;
#pragma unroll
      for (int k = 0; k < kPerLane; ++k) {
        const int e = lane + 64 * k;
        if (e < a.d) out[e] = static_cast<T>(acc[k] * inv);
      }
    }
    if (pair + step >= at.total * a.heads) return;
  }
}

template <typename T, int D, bool PART>
static diopiError_t launchTile(hipStream_t stream, const PtArgs& x, int64_t wgs) {
  constexpr size_t lds = 4 * (size_t)(kPtTile * D) * sizeof(T);
  static_assert(lds >= 4 * 32 * (D + 8) * sizeof(T), "the output has to fit in the stages");
  AMD_HIP(allowDynamicLds(reinterpret_cast<const void*>(&pagedTileKernel<T, D, PART>), (int)lds));
  hipLaunchKernelGGL((pagedTileKernel<T, D, PART>), dim3((unsigned)wgs), dim3(256), lds, stream, x);
  AMD_LAUNCH_CHECK();
  return diopiSuccess;
}

template <int D, bool PART>
static diopiError_t launchFloat(hipStream_t stream, const PtArgs& x, int64_t wgs) {
  constexpr int lds = 4 * 16 * (D + 4) * (int)sizeof(float);
  AMD_HIP(allowDynamicLds(reinterpret_cast<const void*>(&pagedFloatKernel<D, PART>), lds));
  hipLaunchKernelGGL((pagedFloatKernel<D, PART>), dim3((unsigned)wgs), dim3(256), lds, stream, x);
  AMD_LAUNCH_CHECK();
  return diopiSuccess;
}

bool pagedAttentionTiles(const PaArgs& a, diopiDtype_t dtype) {
  const int64_t size = dtypeSize(dtype);
  if (a.d * size % 16 != 0 || a.d > 256 || a.slots > 0x7fffffff) return false;
  const int64_t bits = (int64_t)reinterpret_cast<uintptr_t>(a.k) | (int64_t)reinterpret_cast<uintptr_t>(a.v) | (int64_t)reinterpret_cast<uintptr_t>(a.q) |
                       (int64_t)reinterpret_cast<uintptr_t>(a.out) |
                       (a.kSlotStride | a.kHeadStride | a.vSlotStride | a.vHeadStride | a.qTok | a.qHead | a.oTok | a.oHead) * size;
  if ((bits & 15) != 0 || a.kSlotStride < 0 || a.vSlotStride < 0 || std::max(a.kSlotStride, a.vSlotStride) * size > 0xffffffffll) return false;
  // 32 bits hold the columns of a sequence
  return std::min<int64_t>(a.maxNew, a.rows) * (a.heads / a.kvHeads) < 1 << 30;
}

diopiError_t pagedAttentionMfma(diopiContextHandle_t ctx, hipStream_t stream, const PaArgs& a, diopiDtype_t dtype) {
  PtArgs x{};
  x.a = a;
  const bool wide = dtype == diopi_dtype_float32;
  if (!wide) x.kSlotBytes = (unsigned)(a.kSlotStride * 2), x.vSlotBytes = (unsigned)(a.vSlotStride * 2);
  const int64_t group = a.heads / a.kvHeads, tokens = std::min<int64_t>(a.rows, (int64_t)a.batch * a.maxNew), cus = computeUnits();
  const int64_t tiles = std::max<int64_t>(1, std::min<int64_t>(ceilDiv(a.maxLen, kPtTile), ceilDiv(a.sinks, kPtTile) + ceilDiv((int64_t)a.window + kPtCols, kPtTile)));
  // Blocks of columns: what the rows of q fill, and one partly filled for each sequence at most. Where they leave compute units without
  // work the sequences are walked in shares.
  const int64_t blocks = ceilDiv(tokens * group, wide ? kPtFloatCols : kPtCols), most = blocks + std::min<int64_t>(a.batch, tokens);
  const int64_t perKv = std::max<int64_t>(blocks, std::min<int64_t>(a.batch, tokens));
  int64_t splits = std::max<int64_t>(1, 2 * cus / (perKv * a.kvHeads));
  splits = std::min<int64_t>({splits, kPtMaxSplit, ceilDiv(tiles, 2)});
  x.tilesPerSplit = (int)ceilDiv(tiles, splits);
  x.splits = (int)ceilDiv(tiles, x.tilesPerSplit);
  if (x.splits > 1) {
    void* ws = nullptr;
    AMD_TRY(requireWorkspace(ctx, a.rows * a.heads * x.splits * (2 + a.d) * (int64_t)sizeof(float), &ws));
    x.partial = static_cast<float*>(ws);
  }
  const int64_t wgs = most * x.splits * a.kvHeads;
  AMD_CHECK(wgs < 1 << 24, "paged attention: %ld rows of %d heads exceed the grid limits", (long)a.rows, a.heads);  // (2^32 threads)
#define SIZE_CALL(CALL)               \
  do {                                \
    if (a.d <= 64) CALL(64);          \
    else if (a.d <= 128) CALL(128);   \
    else CALL(256);                   \
  } while (0)
#define BF16_CALL(D) AMD_TRY((a.d == D ? launchTile<bf16_t, D, false>(stream, x, wgs) : launchTile<bf16_t, D, true>(stream, x, wgs)))
#define FP16_CALL(D) AMD_TRY((a.d == D ? launchTile<half_t, D, false>(stream, x, wgs) : launchTile<half_t, D, true>(stream, x, wgs)))
#define FP32_CALL(D) AMD_TRY((a.d == D ? launchFloat<D, false>(stream, x, wgs) : launchFloat<D, true>(stream, x, wgs)))
  if (dtype == diopi_dtype_bfloat16) SIZE_CALL(BF16_CALL);
  else if (dtype == diopi_dtype_float16) SIZE_CALL(FP16_CALL);
  else SIZE_CALL(FP32_CALL);
#undef FP32_CALL
#undef FP16_CALL
#undef BF16_CALL
#undef SIZE_CALL
  if (x.splits > 1) {
    const dim3 grid((unsigned)std::min<int64_t>(ceilDiv(tokens * a.heads, 4), 1 << 23)), block(256);
    if (dtype == diopi_dtype_bfloat16) hipLaunchKernelGGL((pagedMergeKernel<bf16_t, kPtCols>), grid, block, 0, stream, x);
    else if (dtype == diopi_dtype_float16) hipLaunchKernelGGL((pagedMergeKernel<half_t, kPtCols>), grid, block, 0, stream, x);
    else hipLaunchKernelGGL((pagedMergeKernel<float, kPtFloatCols>), grid, block, 0, stream, x);
    AMD_LAUNCH_CHECK();
  }
  return diopiSuccess;
}

}  // namespace amd
