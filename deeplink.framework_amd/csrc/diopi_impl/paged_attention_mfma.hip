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
// Bound by the matrix pipe and the vector ALUs, between which the two waves of a SIMD change places less than they could: bf16, 32 heads of 128, 2 x
// 2048 new tokens behind 6000 555 us, 0.85 PFLOP/s (520 to 555 from card to card and with the same inputs again or others each time), the pipe busy 46 % of
// the time, the ALUs about as long, LDS 24 %. A block spends 8.6 us besides its
// tiles (search 2.3, slots and first tiles 3.7, output 2.6), of which a second workgroup on the compute unit hides a part: prompts of
// 2048 with a window of 512, 11 tiles to a block, 133 us. Heads of 256 leave one workgroup to a compute unit, with some registers spilled: 2 x 1024
// behind 3000, 16 heads, 192 us, 0.61 PFLOP/s.
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
constexpr int kPtFewCols = 32;                    // 16-bit rows: sequences of up to so many columns take the other form

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
  // partial results of blocks of columns: weighted sums of V [rows, heads, splits, d]; maximum and sum [rows, heads, splits]. Rows: see ptPartialRow
  float* partial;
  float2* partialState;
  int splits, tilesPerSplit;
  unsigned kSlotBytes, vSlotBytes;
  float* fewPartial;  // of sequences with few columns: [slices, fewSplits, 2 + d] (see ptFewSlice)
  int16_t fewSplits = 0;
  int16_t fewCols;    // slices of each sequence and K/V head; 0: one for each row of q and head
  int fewChunk = 1;
  int64_t tilePieces;  // workgroups for each K/V head that take blocks of columns
  unsigned tileWgs;    // all of them
  int partialSeq;      // rows of `partial` of each sequence; 0: the rows of q
  int64_t turn;        // see pagedPieces
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

// The tokens that some of the new ones of a sequence with few columns see, in order: the first `sinks`, then from `low` on to the last new one.
// Without a gap between the two, from token 0 on (sinks = 0): the later new tokens' first ones do not end where the first one's window begins.
struct PtList {
  int sinks, low, n;
  __device__ __forceinline__ PtList(const PaArgs& a, const PaSequence& s) {
    low = max(0, s.origin + s.first - a.window + 1);
    if (low <= a.sinks) low = 0;
    sinks = min(a.sinks, low);
    n = sinks + max(0, s.origin + s.end - low);
  }
  __device__ __forceinline__ int token(int i) const { return i < sinks ? i : low + (i - sinks); }
};
__device__ __forceinline__ int ptColumns(const PaArgs& a, const PaSequence& s) {  // (cut where 32 bits end: then there are many)
  return (int)min((int64_t)(s.end - s.first) * a.group, (int64_t)1 << 30);
}
__device__ __forceinline__ int ptFewShares(const PtArgs& x, const PaSequence& s) {
  return max(1, (PtList(x.a, s).n + x.fewChunk - 1) / x.fewChunk);
}

// Blocks of columns of a sequence, and the most shares that one of them has.
template <int COLS>
struct PtPieces {
  int blocks, splits;
  __device__ __forceinline__ PtPieces(const PtArgs& x, const PaSequence& s) {
    const int group = x.a.group, tokens = s.end - s.first;
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

// Where partial results have the `at`th new token of sequence b that has a row in q. A row of q for each, or, where q has more rows than the
// sequences can have new tokens (rows of no sequence, as in a recorded call for up to so many tokens), so many for each sequence.
__device__ __forceinline__ int64_t ptPartialRow(const PtArgs& x, const PaSequence& s, int b, int at) {
  return x.partialSeq != 0 ? (int64_t)b * x.partialSeq + at : s.start + s.first + at;
}
// The same for column `col` of a sequence with few of them.
__device__ __forceinline__ int64_t ptFewSlice(const PtArgs& x, const PaSequence& s, int b, int kvh, int col) {
  if (x.fewCols != 0) return ((int64_t)b * x.a.kvHeads + kvh) * x.fewCols + col;
  const int at = paOfGroup(x.a, col);
  return (s.start + s.first + at) * x.a.heads + kvh * x.a.group + (col - at * x.a.group);
}

// Column `col` of a piece of work by itself, on the vector ALUs of one wave.
template <typename T, int D>
__device__ __forceinline__ void pagedAgain(const PtArgs& x, const PaSequence& s, int b, int kvh, int64_t locBase, const PtSpan& span, int t0, int t1, int split,
                                           bool whole, int col) {
  const PaArgs& a = x.a;
  const int lane = threadIdx.x & 63, group = a.group, at = paOfGroup(a, col), token = s.first + at, h = kvh * group + (col - at * group), p = s.origin + token;
  const int64_t row = s.start + token;
  int head, low;
  paSeen(a, p, &head, &low);
  // of the tiles' tokens those that it sees: of the first ones, and of the others
  const int from = span.base(max(t0, span.sinkTiles)), to = t1 > span.sinkTiles ? min(span.base(t1), p + 1) : 0;
  const int first0 = span.sinkTiles > 0 ? min(t0, span.sinkTiles) * kPtTile : from, first1 = span.sinkTiles > 0 ? min(head, min(t1, span.sinkTiles) * kPtTile) : min(head, to);
  PaColumn<T, D / 64, (D > 128 ? 4 : 8)> one;
  one.walk(a, reinterpret_cast<const T*>(a.q) + row * a.qTok + (int64_t)h * a.qHead, kvh, locBase, first0, first1, max(from, low), to, 0, 64);
  const int64_t slice = (ptPartialRow(x, s, b, at) * a.heads + h) * x.splits + split;
  float* dst = x.partial + slice * a.d;
  T* out = reinterpret_cast<T*>(a.out) + row * a.oTok + (int64_t)h * a.oHead;
  const float inv = one.l == 0.f ? 0.f : 1.f / one.l;
  if (!whole && lane == 0) x.partialState[slice] = float2{one.m, one.l};
#pragma unroll
  for (int j = 0; j < D / 64; ++j) {
    const int e = lane + 64 * j;
    if (e >= a.d) continue;
    if (whole) out[e] = static_cast<T>(one.acc[j] * inv);
    else dst[e] = one.acc[j];
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
  extern __shared__ __attribute__((aligned(1024))) char ptSmem[];  // (the fragments' addresses are put together by XOR)
  const PaArgs& a = x.a;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l31 = lane & 31, half = lane >> 5;
  const int group = a.group, cols = (s.end - s.first) * group, c0 = block * kPtCols + wave * 32;
  const bool waveLives = c0 < cols;
  const int col = min(c0 + l31, cols - 1), mine = paOfGroup(a, col), token = s.first + mine, h = kvh * group + (col - mine * group);
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
    if (t >= t1) return int2{0, 0};
    return paAsk(a.bLoc, locBase + min(span.base(t) + lane, span.limit(t) - 1), a.loc64);
  };
  auto inPool = [&](int2 asked) {
    const int64_t slot = paIndex(asked, a.loc64);
    return slot >= 0 && slot < a.slots;
  };
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
  auto rowsOf = [&](int2 asked, uint64_t in, int (&rows)[NLD]) {
    const int instead = in != 0 ? __builtin_amdgcn_readlane(asked.x, __builtin_ctzll(in)) : 0;
    const int mine = inPool(asked) ? asked.x : instead;
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
  int2 asked;                             // slots of tile t + 3
  {
    const int2 first = askSlot(t0), second = askSlot(t0 + 1), third = askSlot(t0 + 2);
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
    if (half == 0 && c0 + l31 < cols && (again >> l31 & 1) == 0) x.partialState[(ptPartialRow(x, s, b, mine) * a.heads + h) * x.splits + split] = float2{m - M::kRaise, l};
    // half of a column's elements at a time through LDS, so that a row of workspace is written in whole pieces
    constexpr int kHalf = D / 2, OF = kHalf + 4, PER = kHalf / 4;  // floats of a padded row; pieces of 16 bytes
    float* sO = reinterpret_cast<float*>(ptSmem) + wave * 32 * OF;
#pragma unroll
    for (int pass = 0; pass < 2; ++pass) {
      exchangeInWave();
#pragma unroll
      for (int dt = 0; dt < DT / 2; ++dt)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const f32x16& part = o[pass * (DT / 2) + dt];
          *reinterpret_cast<f32x4*>(sO + l31 * OF + dt * 32 + g * 8 + half * 4) = f32x4{part[g * 4], part[g * 4 + 1], part[g * 4 + 2], part[g * 4 + 3]};
        }
      exchangeInWave();
#pragma unroll
      for (int i = 0; i < 32 * PER / 64; ++i) {
        const int piece = lane + 64 * i, r = piece / PER, e = (piece % PER) * 4, oc = c0 + r;
        if (oc >= cols || (again >> r & 1) != 0 || (PART && pass * kHalf + e >= a.d)) continue;
        const int at = paOfGroup(a, oc);
        const int64_t to = ptPartialRow(x, s, b, at) * a.heads + kvh * group + (oc - at * group);
        *reinterpret_cast<f32x4*>(x.partial + (to * x.splits + split) * a.d + pass * kHalf + e) = *reinterpret_cast<const f32x4*>(sO + r * OF + e);
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
      const int oc = c0 + r, at = paOfGroup(a, oc), tok = s.first + at;
      if (oc < cols && (again >> r & 1) == 0 && (!PART || c * 8 < a.d))
        *reinterpret_cast<Frag*>(reinterpret_cast<T*>(a.out) + (s.start + tok) * a.oTok + (int64_t)(kvh * group + (oc - at * group)) * a.oHead + c * 8) =
            *reinterpret_cast<const Frag*>(sO + r * OS + c * 8);
  }
  }
  for (; again != 0; again &= again - 1) pagedAgain<T, D>(x, s, b, kvh, locBase, span, t0, t1, split, whole, c0 + __builtin_ctz(again));
}

// A workgroup's pieces of work, from a list for each K/V head: sequence after sequence, shares from the first, blocks from the last, which has
// the most tiles. x.tilePieces workgroups for each K/V head, the number of pieces unless sequences share rows of q; sequences of up to FEW
// columns are not among them.
// Where all of them run at once, two to a compute unit, the second round of units (from x.turn pieces on) goes through the rest of the list
// from its end: a block with many tiles runs next to one with few.
template <int COLS, int FEW, typename F>
__device__ __forceinline__ void pagedPieces(const PtArgs& x, F&& walk) {
  const PaArgs& a = x.a;
  const int kvh = blockIdx.x % a.kvHeads, group = a.group;
  const int64_t step = x.tilePieces, mine = blockIdx.x / a.kvHeads;
  for (int64_t u = mine < x.turn ? mine : step - 1 - (mine - x.turn);; u += step) {
    const PaPlace at = paFind(a, u, [&](const PaSequence& s) { return ptColumns(a, s) <= FEW ? 0 : PtPieces<COLS>(x, s).all(); });
    if (at.b < 0) return;
    const PaSequence& s = at.s;
    const PtPieces<COLS> pieces(x, s);
    const int split = at.at / pieces.blocks, block = pieces.blocks - 1 - at.at % pieces.blocks;
    const int cols = (s.end - s.first) * group, origin = s.origin + s.first;
    const PtSpan span(a, origin + paOfGroup(a, block * COLS), origin + paOfGroup(a, min(block * COLS + COLS - 1, cols - 1)));
    const bool whole = span.tiles <= x.tilesPerSplit;
    const int t0 = split * x.tilesPerSplit, t1 = min(span.tiles, t0 + x.tilesPerSplit);
    if (split == 0 || t0 < span.tiles) walk(s, at.b, kvh, block, span, t0, t1, split, whole);
    if (u + step >= at.total) return;
    __syncthreads();  // (the next piece's tiles take the place of this one's output)
  }
}

// ---------------------------------------------------------------- few columns --
// Sequences with up to 32 columns of a K/V head (a token or a few speculated ones): bound by memory. A workgroup takes a share of the
// tokens and its waves cut that, each with a two-stage LDS ring of its own: no barriers until their states meet. With WIDE a
// wave takes all tokens of a K/V head and the workgroup four heads, for sequences so short that a wave's share would be nothing.
//   * S^T = K . Q^T (16x16x32), 16 tokens x 16 columns at a time: a lane holds four tokens' scores of one column, and its probabilities
//     are as they lie the operand P^T of O^T += V^T . P^T, whose 32 places hold the 16 tokens twice: with the rounded
//     probability and with what the rounding left, which makes 16 bits of it in bf16 and 22 in fp16 at no cost.
//   * the tokens that are seen are a list without gaps (PtList); their slots are looked up 128 at a time.
// bf16, heads of 128: 64 x 1 new token behind 2048, 32 heads 340 us, 6.3 TB/s; 1 x 5 behind 1777, 32 heads on 8, a chain of loads, 8.6 us and 4 for
// the launch that joins the shares.
//   * the running maximum is replaced only when a score exceeds it by more than 2^8.
constexpr int kPfWaves = 4, kPfTile = 16, kPfBlock = 128, kPfStages = 2;
template <typename T>
struct PfMfma;
template <>
struct PfMfma<bf16_t> {
  static __device__ __forceinline__ f32x4 run(bf16x8 a, bf16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
};
template <>
struct PfMfma<half_t> {
  static __device__ __forceinline__ f32x4 run(f16x8 a, f16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
};
// XOR on the 16-byte piece index of row r in LDS: 16 rows' pieces of one index (K), the 8 rows x 32 bytes of half a transposing read (V)
// fall on different banks.
template <int D>
__device__ __forceinline__ int pfSwizzleK(int r) { return D >= 128 ? (r & 15) : ((r >> 1) & 7); }
template <int D>
__device__ __forceinline__ int pfSwizzleV(int r) { return D >= 128 ? 2 * (r & 7) : 2 * ((r >> 1) & 3); }

template <int N>
__device__ __forceinline__ void waitLoadsBut() {  // all but the wave's N youngest vector-memory operations are done
  asm volatile("s_waitcnt vmcnt(%0)" : : "n"(N) : "memory");
}

// CT: tiles of 16 columns, 1 or 2. (As a variant and not a branch around the second one's products: of products that are branched around
// the compiler, hipcc 7.2, has read the result before it was there.)
template <typename T, int D, bool WIDE, int CT>
__device__ __forceinline__ void pagedFewBlock(const PtArgs& x, const PaSequence& s, int b, int kvh, int split) {
  using Frag = typename PtMfma<T>::Frag;
  using Half = typename PtMfma<T>::Half;
  constexpr int ROWB = D * 2, CPR = D / 8, RPL = 64 / CPR, NLD = kPfTile / RPL, KS = D / 32, DT = D / 16;
  constexpr unsigned kMatBytes = kPfTile * ROWB, kStageBytes = 2 * kMatBytes;
  constexpr float kRaise = PtMfma<T>::kRaise;
  extern __shared__ __attribute__((aligned(1024))) char ptSmem[];  // (the fragments' addresses are put together by XOR)
  __shared__ int slotBuf[kPfWaves][kPfBlock];
  __shared__ float stateBuf[kPfWaves][2][kPtFewCols];
  __shared__ int again[kPtFewCols];
  const PaArgs& a = x.a;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), c16 = lane & 15, quad = lane >> 4;
  const int group = a.group, cols = (s.end - s.first) * group;
  const PtList list(a, s);
  const int64_t locBase = (int64_t)b * a.locRowStride + (a.maxLen - s.len);
  const int chunkBegin = split * x.fewChunk, chunkEnd = min(list.n, chunkBegin + x.fewChunk);
  const int share = WIDE ? chunkEnd - chunkBegin : ((chunkEnd - chunkBegin + kPfWaves - 1) / kPfWaves + kPfTile - 1) / kPfTile * kPfTile;
  const int from = WIDE ? chunkBegin : chunkBegin + wave * share, to = min(chunkEnd, from + share);

  // slots of a block of tokens, past the last one that again; the first block's are asked for before the rows of q: loads come back in order
  int2 raw[kPfBlock / 64];
  auto askSlots = [&](int b0) {
    const int cnt = min(kPfBlock, to - b0);
#pragma unroll
    for (int i = 0; i < kPfBlock / 64; ++i) raw[i] = paAsk(a.bLoc, locBase + list.token(b0 + min(i * 64 + lane, cnt - 1)), a.loc64);
  };
  if (from < to) askSlots(from);
  Frag qf[CT][KS];
  int p[CT], sinksSeen[CT];
#pragma unroll
  for (int ct = 0; ct < CT; ++ct) {
    const int col = min(ct * 16 + c16, cols - 1), at = paOfGroup(a, col), token = s.first + at;
    p[ct] = s.origin + token, sinksSeen[ct] = max(0, min(a.sinks, p[ct] + 1));
    const T* q = reinterpret_cast<const T*>(a.q) + (s.start + token) * a.qTok + (int64_t)(kvh * group + (col - at * group)) * a.qHead;
#pragma unroll
    for (int k = 0; k < KS; ++k) {
      const int e = 32 * k + 8 * quad;
      qf[ct][k] = *reinterpret_cast<const Frag*>(q + (e < a.d ? e : 0));
      if (e >= a.d) {
#pragma unroll
        for (int j = 0; j < 8; ++j) qf[ct][k][j] = static_cast<T>(0.f);
      }
    }
  }
  const int pMin = s.origin + s.first, pMax = s.origin + s.end - 1, window = a.window;
  f32x4 acc[CT][DT];
  float m[CT], l[CT];
#pragma unroll
  for (int ct = 0; ct < CT; ++ct) {
    m[ct] = -INFINITY, l[ct] = 0.f;
#pragma unroll
    for (int d = 0; d < DT; ++d) acc[ct][d] = f32x4{0.f, 0.f, 0.f, 0.f};
  }

  // ring: load i of a matrix fills rows i * RPL ... of its tile, lane (row lane / CPR of those, piece lane % CPR) with the piece that the swizzle
  // puts there; behind a row's end the first piece again, which meets zeros of q or gives places that are not stored
  const unsigned ring = (unsigned)(uintptr_t)ptSmem + (unsigned)wave * (kPfStages * kStageBytes);
  int kOff[NLD], vOff[NLD];
#pragma unroll
  for (int i = 0; i < NLD; ++i) {
    const int row = i * RPL + lane / CPR, piece = lane % CPR, kc = piece ^ pfSwizzleK<D>(row), vc = piece ^ pfSwizzleV<D>(row);
    kOff[i] = kc * 8 < a.d ? kc * 16 : 0, vOff[i] = vc * 8 < a.d ? vc * 16 : 0;
  }
  const char* const kBase = reinterpret_cast<const char*>(reinterpret_cast<const T*>(a.k) + kvh * a.kHeadStride);
  const char* const vBase = reinterpret_cast<const char*>(reinterpret_cast<const T*>(a.v) + kvh * a.vHeadStride);
  int* const slots = slotBuf[wave];
  auto issue = [&](int tile, int stage) {
    const unsigned at = ring + (unsigned)stage * kStageBytes;
    unsigned slot[NLD];
#pragma unroll
    for (int i = 0; i < NLD; ++i) slot[i] = (unsigned)slots[tile * kPfTile + i * RPL + lane / CPR] & 0x7fffffffu;
#pragma unroll
    for (int i = 0; i < NLD; ++i) globalLoadToLds16Stream(kBase + ((uint64_t)slot[i] * x.kSlotBytes + (unsigned)kOff[i]), at + i * 1024u);
#pragma unroll
    for (int i = 0; i < NLD; ++i) globalLoadToLds16Stream(vBase + ((uint64_t)slot[i] * x.vSlotBytes + (unsigned)vOff[i]), at + kMatBytes + i * 1024u);
  };

  for (int b0 = from; b0 < to; b0 += kPfBlock) {
    const int cnt = min(kPfBlock, to - b0), tiles = (cnt + kPfTile - 1) / kPfTile;
    // a slot outside the pool is skipped, never dereferenced: it is marked by its top bit, and another of the block stands in (slot 0
    // where there is none)
    uint64_t in[kPfBlock / 64];
    if (b0 != from) askSlots(b0);
    int instead = 0;
#pragma unroll
    for (int i = 0; i < kPfBlock / 64; ++i) {
      const int64_t slot = paIndex(raw[i], a.loc64);
      in[i] = __builtin_amdgcn_ballot_w64(slot >= 0 && slot < a.slots);
      if (in[i] != 0) instead = __builtin_amdgcn_readlane(raw[i].x, __builtin_ctzll(in[i]));
    }
#pragma unroll
    for (int i = 0; i < kPfBlock / 64; ++i) slots[i * 64 + lane] = in[i] >> lane & 1 ? raw[i].x : (int)(0x80000000u | (unsigned)instead);
    const bool skips = (in[0] & in[1]) != ~0ull;
    static_assert(kPfBlock == 128, "two words of 64 slots");
    exchangeInWave();
    // (also the reads of the block before: the ring's loads overwrite what they read)
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" : : : "memory");
    issue(0, 0);
    for (int t = 0; t < tiles; ++t) {
      const int stage = t & 1;
      if (t + 1 < tiles) {
        // the tile read last in the other stage has been consumed: its reads are done before the loads that overwrite it go out
        asm volatile("s_waitcnt lgkmcnt(0)" : : : "memory");
        issue(t + 1, stage ^ 1);
        waitLoadsBut<2 * NLD>();
      } else {
        waitLoadsBut<0>();
      }
      const unsigned at = ring + (unsigned)stage * kStageBytes;
      typedef __attribute__((address_space(3))) const Frag* LdsFrag;
      typedef __attribute__((address_space(3))) s16x4* LdsTr;
      const int v0 = b0 + t * kPfTile, last = v0 + kPfTile - 1;
      // whether every column sees all of the tile (uniform)
      const bool all = !skips && last < to && list.token(last) <= pMin && (list.token(v0) > pMax - window || list.token(last) < a.sinks);
      f32x4 sc[CT][2];
#pragma unroll
      for (int ct = 0; ct < CT; ++ct) sc[ct][0] = sc[ct][1] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int k = 0; k < KS; ++k) {
        const Frag kf = *(LdsFrag)(uintptr_t)(at + (unsigned)(c16 * ROWB + (((4 * k + quad) ^ pfSwizzleK<D>(c16)) << 4)));
#pragma unroll
        for (int ct = 0; ct < CT; ++ct) sc[ct][k & 1] = PfMfma<T>::run(kf, qf[ct][k], sc[ct][k & 1]);
      }
      Frag pr[CT];
#pragma unroll
      for (int ct = 0; ct < CT; ++ct) {
        float w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = (sc[ct][0][i] + sc[ct][1][i]) * a.scaleLog2e;
        if (!all) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int v = v0 + 4 * quad + i, kj = list.token(v);
            const bool sees = v < to && ((unsigned)(p[ct] - kj) < (unsigned)window || kj < sinksSeen[ct]) && slots[t * kPfTile + 4 * quad + i] >= 0;
            if (!sees) w[i] = -INFINITY;
          }
        }
        float mt = fmaxf(fmaxf(w[0], w[1]), fmaxf(w[2], w[3]));
        if (__builtin_amdgcn_ballot_w64(mt > m[ct] + kPtRescaleStep || (m[ct] == -INFINITY && mt != -INFINITY)) != 0) {
          auto sw = __builtin_amdgcn_permlane32_swap(__float_as_uint(mt), __float_as_uint(mt), false, false);
          mt = fmaxf(__uint_as_float(sw[0]), __uint_as_float(sw[1]));
          sw = __builtin_amdgcn_permlane16_swap(__float_as_uint(mt), __float_as_uint(mt), false, false);
          mt = fmaxf(__uint_as_float(sw[0]), __uint_as_float(sw[1]));
          if (mt > m[ct]) {
            const float corr = __builtin_amdgcn_exp2f(m[ct] - mt);  // no maximum yet: 0, and the sums are 0
            m[ct] = mt, l[ct] *= corr;
#pragma unroll
            for (int d = 0; d < DT; ++d)
#pragma unroll
              for (int i = 0; i < 4; ++i) acc[ct][d][i] *= corr;
          }
        }
        const float ref = m[ct] == -INFINITY ? 0.f : m[ct];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float e = __builtin_amdgcn_exp2f(behindRounded(w[i], ref) + kRaise);
          l[ct] += e;
          const T hi = static_cast<T>(e);
          pr[ct][i] = hi, pr[ct][4 + i] = static_cast<T>(e - static_cast<float>(hi));
        }
      }
      const int row = 4 * quad + (c16 >> 2);
      const unsigned vRow = at + kMatBytes + (unsigned)(row * ROWB + (lane & 1) * 8);
#pragma unroll
      for (int d = 0; d < DT; ++d) {
        const unsigned piece = (unsigned)((2 * d + ((lane & 3) >> 1)) ^ pfSwizzleV<D>(row)) << 4;
        const u32x2 v = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsTr)(uintptr_t)(vRow + piece)));
        const Frag vf = __builtin_bit_cast(Frag, u32x4{v[0], v[1], v[0], v[1]});
#pragma unroll
        for (int ct = 0; ct < CT; ++ct) acc[ct][d] = PfMfma<T>::run(vf, pr[ct], acc[ct][d]);
      }
    }
  }

  // ---- the states: every lane group holds its own share of l
  float lowered = 1.f;  // (what raised probabilities have to be divided by)
  if (kRaise != 0.f) lowered = 1.f / (1 << (int)kRaise);
#pragma unroll
  for (int ct = 0; ct < CT; ++ct) {
    auto sw = __builtin_amdgcn_permlane32_swap(__float_as_uint(l[ct]), __float_as_uint(l[ct]), false, false);
    l[ct] = __uint_as_float(sw[0]) + __uint_as_float(sw[1]);
    sw = __builtin_amdgcn_permlane16_swap(__float_as_uint(l[ct]), __float_as_uint(l[ct]), false, false);
    l[ct] = __uint_as_float(sw[0]) + __uint_as_float(sw[1]);
    l[ct] *= lowered;
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[ct][d][i] *= lowered;
  }
  const int shares = ptFewShares(x, s);
  const bool whole = shares == 1;
  // where column `col` of this K/V head goes, 4 elements from e on, from sums against the maximum
  auto store = [&](int col, int e, float mCol, float lCol, f32x4 o) {
    const int at = paOfGroup(a, col), token = s.first + at;
    if (whole) {
      const float inv = lCol > 0.f ? 1.f / lCol : 0.f;
      Half r;
#pragma unroll
      for (int i = 0; i < 4; ++i) r[i] = static_cast<T>(o[i] * inv);
      *reinterpret_cast<Half*>(reinterpret_cast<T*>(a.out) + (s.start + token) * a.oTok + (int64_t)(kvh * group + (col - at * group)) * a.oHead + e) = r;
    } else {
      float* dst = x.fewPartial + (ptFewSlice(x, s, b, kvh, col) * x.fewSplits + split) * (2 + a.d);
      if (e == 0) dst[0] = mCol, dst[1] = lCol;
      *reinterpret_cast<float2*>(dst + 2 + e) = float2{o[0], o[1]};
      *reinterpret_cast<float2*>(dst + 4 + e) = float2{o[2], o[3]};
    }
  };
  auto finite = [](float v) { return fabsf(v) < INFINITY; };
  // a column whose sums are not finite: again by itself, the tokens that it sees alone (one wave)
  auto walkAgain = [&](int col) {
    const int at = paOfGroup(a, col), token = s.first + at, h = kvh * group + (col - at * group);
    int head, low;
    paSeen(a, s.origin + token, &head, &low);
    // of the share's tokens those that it sees
    const int first0 = min(chunkBegin, list.sinks), first1 = min(head, min(chunkEnd, list.sinks));
    const int next0 = list.low + max(0, chunkBegin - list.sinks), next1 = list.low + max(0, chunkEnd - list.sinks);
    const int more1 = list.sinks == 0 ? min(head, next1) : 0;  // (without a list of first tokens apart they lie in the other part)
    PaColumn<T, D / 64, (D > 128 ? 4 : 8)> one;
    const T* q = reinterpret_cast<const T*>(a.q) + (s.start + token) * a.qTok + (int64_t)h * a.qHead;
    one.walk(a, q, kvh, locBase, list.sinks == 0 ? next0 : first0, list.sinks == 0 ? more1 : first1, max(next0, low), min(next1, s.origin + token + 1), 0, 64);
    const float inv = one.l == 0.f ? 0.f : 1.f / one.l;
    T* out = reinterpret_cast<T*>(a.out) + (s.start + token) * a.oTok + (int64_t)h * a.oHead;
    float* dst = x.fewPartial + (ptFewSlice(x, s, b, kvh, col) * x.fewSplits + split) * (2 + a.d);
    if (!whole && lane == 0) dst[0] = one.m, dst[1] = one.l;
#pragma unroll
    for (int j = 0; j < D / 64; ++j) {
      const int e = lane + 64 * j;
      if (e >= a.d) continue;
      if (whole) out[e] = static_cast<T>(one.acc[j] * inv);
      else dst[2 + e] = one.acc[j];
    }
  };
  if (WIDE) {
    uint32_t bad = 0;
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) {
      bool odd = !finite(l[ct]);
#pragma unroll
      for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int i = 0; i < 4; ++i) odd |= !finite(acc[ct][d][i]);
      const uint64_t lanes = __builtin_amdgcn_ballot_w64(odd && ct * 16 + c16 < cols);
      const uint32_t sixteen = (uint32_t)((lanes | lanes >> 16 | lanes >> 32 | lanes >> 48) & 0xffffu);
      bad |= sixteen << (16 * ct);
      if (ct * 16 + c16 < cols && (sixteen >> c16 & 1) == 0) {
#pragma unroll
        for (int d = 0; d < DT; ++d)
          if (16 * d + 4 * quad < a.d) store(ct * 16 + c16, 16 * d + 4 * quad, m[ct], l[ct], acc[ct][d]);
      }
    }
    for (; bad != 0; bad &= bad - 1) walkAgain(__builtin_ctz(bad));
    return;
  }
  // waves meet in LDS, a tile of 16 columns at a time (without a wait for what has been stored: 1 us)
  auto meet = []() {
    asm volatile("s_waitcnt lgkmcnt(0)" : : : "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" : : : "memory");
  };
  constexpr int kRedRow = D + 4;
  float* const red = reinterpret_cast<float*>(ptSmem);  // the ring: every load into it has been waited for
  if (threadIdx.x < kPtFewCols) again[threadIdx.x] = 0;
#pragma unroll
  for (int ct = 0; ct < CT; ++ct)
    if (quad == 0) stateBuf[wave][0][ct * 16 + c16] = m[ct], stateBuf[wave][1][ct * 16 + c16] = l[ct];
#pragma unroll
  for (int ct = 0; ct < CT; ++ct) {
    meet();
#pragma unroll
    for (int d = 0; d < DT; ++d) *reinterpret_cast<f32x4*>(red + (wave * 16 + c16) * kRedRow + 16 * d + 4 * quad) = acc[ct][d];
    meet();
    const int here = min(16, cols - ct * 16);
    for (int i = threadIdx.x; i < here * (D / 4); i += kPfWaves * 64) {
      const int j = i / (D / 4), e = (i % (D / 4)) * 4, col = ct * 16 + j;
      if (e >= a.d) continue;
      float mAll = -INFINITY, lAll = 0.f;
#pragma unroll
      for (int k = 0; k < kPfWaves; ++k) mAll = fmaxf(mAll, stateBuf[k][0][col]);
      f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int k = 0; k < kPfWaves; ++k) {
        const float mk = stateBuf[k][0][col], w = mk == -INFINITY ? 0.f : exp2f(mk - mAll);
        lAll += stateBuf[k][1][col] * w;
        const f32x4 v = *reinterpret_cast<const f32x4*>(red + (k * 16 + j) * kRedRow + e);
#pragma unroll
        for (int c = 0; c < 4; ++c) o[c] += v[c] * w;
      }
      bool odd = !finite(lAll);
#pragma unroll
      for (int c = 0; c < 4; ++c) odd |= !finite(o[c]);
      if (odd) again[col] = 1;
      else store(col, e, mAll, lAll, o);
    }
  }
  meet();
  if (__builtin_amdgcn_ballot_w64(again[lane & (kPtFewCols - 1)] != 0) == 0) return;  // (the same for all waves)
  asm volatile("s_waitcnt vmcnt(0)" : : : "memory");  // (pieces of such a column may have been stored by other waves)
  __syncthreads();
  for (int col = wave; col < cols; col += kPfWaves)
    if (again[col] != 0) walkAgain(col);
}

// Piece u of the sequences of few columns: sequence after sequence, shares from the first.
template <typename T, int D, bool WIDE>
__device__ __forceinline__ void pagedFewPiece(const PtArgs& x, int64_t u, int kvh) {
  const PaPlace at = paFind(x.a, u, [&](const PaSequence& s) {
    const int cols = ptColumns(x.a, s);
    return cols == 0 || cols > kPtFewCols ? 0 : ptFewShares(x, s);
  });
  if (at.b < 0) return;
  if (ptColumns(x.a, at.s) <= 16) pagedFewBlock<T, D, WIDE, 1>(x, at.s, at.b, kvh, at.at);
  else pagedFewBlock<T, D, WIDE, 2>(x, at.s, at.b, kvh, at.at);
}

// Sequences of few columns alone. grid: K/V heads (WIDE: groups of four) fastest.
template <typename T, int D, bool WIDE>
__global__ __launch_bounds__(kPfWaves * 64, D > 128 ? 1 : 2) void pagedFewKernel(PtArgs x) {
  const int groups = WIDE ? x.a.kvHeads / kPfWaves : x.a.kvHeads, g = (int)(blockIdx.x % groups);
  pagedFewPiece<T, D, WIDE>(x, blockIdx.x / groups, WIDE ? g * kPfWaves + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) : g);
}

// Sequences of any number of columns: the first x.tileWgs workgroups take blocks of many, the others few.
template <typename T, int D, bool PART>
__global__ __launch_bounds__(256, D > 128 ? 1 : 2) void pagedTileKernel(PtArgs x) {
  if (blockIdx.x >= x.tileWgs) {
    const unsigned i = blockIdx.x - x.tileWgs;
    pagedFewPiece<T, D, false>(x, i / x.a.kvHeads, (int)(i % x.a.kvHeads));
    return;
  }
  pagedPieces<kPtCols, kPtFewCols>(x, [&](const PaSequence& s, int b, int kvh, int block, const PtSpan& span, int t0, int t1, int split, bool whole) {
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
// NC tiles of 16 columns share the rows in registers. G: groups of four waves, which take tiles by turns. 16 x (1 .. 40) new tokens behind 0 .. 260, 8 heads of 64 11 us, latency; 2 x 700 behind 300, 32
// heads of 128 264 us, 56 TFLOP/s: a wave's products wait for its softmax (16 heads of 256, with spilled registers, 401 us, 37 TFLOP/s).
constexpr int kPtFloatCols = 16;
template <int D, bool PART, int NC, int G>
__device__ __forceinline__ void pagedFloatBlock(const PtArgs& x, const PaSequence& s, int b, int kvh, int block, const PtSpan& span, int t0, int t1, int split,
                                                bool whole) {
  constexpr int S = D / 4, E = D / 16, PITCH = D + 4, COLS = kPtFloatCols * NC, WAVES = 4 * G;
  extern __shared__ __attribute__((aligned(1024))) char ptSmem[];
  float* const so = reinterpret_cast<float*>(ptSmem);  // [WAVES][COLS][PITCH]
  __shared__ float sm[WAVES][COLS], sl[WAVES][COLS];
  const PaArgs& a = x.a;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), part = wave & 3, c = lane & 15, g = lane >> 4;
  const int group = a.group, cols = (s.end - s.first) * group, c0 = block * COLS;
  const int64_t locBase = (int64_t)b * a.locRowStride + (a.maxLen - s.len);
  const float* const kHead = reinterpret_cast<const float*>(a.k) + kvh * a.kHeadStride;
  const float* const vHead = reinterpret_cast<const float*>(a.v) + kvh * a.vHeadStride;
  f32x4 qf[NC][S / 4], kf[2][S / 4], vf[2][4][E / 4], o[NC][E];
  int p[NC], sinksSeen[NC];
  // (PART: places past the row's end read its first piece, are zeros in q and K, and give elements that are not stored)
  auto at = [&](int e) { return !PART || e < a.d ? e : 0; };
#pragma unroll
  for (int n = 0; n < NC; ++n) {
    const int col = min(c0 + 16 * n + c, cols - 1), place = paOfGroup(a, col), token = s.first + place, h = kvh * group + (col - place * group);
    p[n] = s.origin + token, sinksSeen[n] = max(0, min(a.sinks, p[n] + 1));
    const float* q = reinterpret_cast<const float*>(a.q) + (s.start + token) * a.qTok + (int64_t)h * a.qHead;
#pragma unroll
    for (int i = 0; i < S / 4; ++i) {
      qf[n][i] = *reinterpret_cast<const f32x4*>(q + at(g * S + 4 * i));
      if (PART && g * S + 4 * i >= a.d) qf[n][i] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
  }
  const int pFirst = __builtin_amdgcn_readlane(p[0], 0), pLast = __builtin_amdgcn_readlane(p[NC - 1], 15), window = a.window;
  auto askSlot = [&](int t) {
    if (t >= t1) return int2{0, 0};
    return paAsk(a.bLoc, locBase + min(span.base(t) + 16 * part + c, span.limit(t) - 1), a.loc64);
  };
  uint32_t valid[2];
  auto fetch = [&](int2 asked, auto buf) {
    constexpr int B = decltype(buf)::value;
    const int64_t slot = paIndex(asked, a.loc64);
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
  float m[NC], l[NC];  // m: in units of log2
#pragma unroll
  for (int n = 0; n < NC; ++n) {
    m[n] = -INFINITY, l[n] = 0.f;
#pragma unroll
    for (int i = 0; i < E; ++i) o[n][i] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  auto tile = [&](int t, auto buf) {
    constexpr int B = decltype(buf)::value;
    const int k0 = span.base(t) + 16 * part;
    if (k0 > pLast || k0 >= span.limit(t) || (k0 + 15 <= pFirst - window && k0 >= a.sinks)) return;  // (uniform: nobody sees any of it)
    f32x4 acc[NC][2];  // two chains each: half the dependent latency
#pragma unroll
    for (int n = 0; n < NC; ++n) acc[n][0] = acc[n][1] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < S; ++i)
#pragma unroll
      for (int n = 0; n < NC; ++n) acc[n][i & 1] = __builtin_amdgcn_mfma_f32_16x16x4f32(kf[B][i >> 2][i & 3], qf[n][i >> 2][i & 3], acc[n][i & 1], 0, 0, 0);
    float w[NC][4];
#pragma unroll
    for (int n = 0; n < NC; ++n) {
      float mx = m[n];
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int kj = k0 + 4 * g + r;
        const bool sees = ((unsigned)(p[n] - kj) < (unsigned)window || kj < sinksSeen[n]) && (valid[B] >> (4 * g + r) & 1) != 0;
        w[n][r] = sees ? (acc[n][0][r] + acc[n][1][r]) * a.scaleLog2e : -INFINITY;
        mx = fmaxf(mx, w[n][r]);
      }
      mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
      mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
      const float ref = mx == -INFINITY ? 0.f : mx, keep = exp2f(m[n] - ref);
      m[n] = mx, l[n] *= keep;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        w[n][r] = exp2f(behindRounded(w[n][r], ref));
        l[n] += w[n][r];
      }
#pragma unroll
      for (int i = 0; i < E; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) o[n][i][r] *= keep;
    }
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int i = 0; i < E; ++i)
#pragma unroll
        for (int n = 0; n < NC; ++n) o[n][i] = __builtin_amdgcn_mfma_f32_16x16x4f32(vf[B][r][i >> 2][i & 3], w[n][r], o[n][i], 0, 0, 0);
  };
  using B0 = std::integral_constant<int, 0>;
  using B1 = std::integral_constant<int, 1>;
  const int tFirst = t0 + (wave >> 2);
  if (tFirst < t1) {
    const int2 first = askSlot(tFirst);
    int2 next = askSlot(tFirst + G);
    fetch(first, B0{});
    for (int t = tFirst; t < t1; t += 2 * G) {
      if (t + G < t1) {
        const int2 slot = next;
        next = askSlot(t + 2 * G);
        fetch(slot, B1{});
      }
      tile(t, B0{});
      if (t + G >= t1) break;
      if (t + 2 * G < t1) {
        const int2 slot = next;
        next = askSlot(t + 3 * G);
        fetch(slot, B0{});
      }
      tile(t + G, B1{});
    }
  }
#pragma unroll
  for (int n = 0; n < NC; ++n) {
    l[n] += __shfl_xor(l[n], 16, 64);
    l[n] += __shfl_xor(l[n], 32, 64);
    if (l[n] != l[n] && m[n] == -INFINITY) m[n] = 0.f;  // scores that are not numbers alone: as a maximum of minus infinity they would be left out
    if (g == 0) sm[wave][16 * n + c] = m[n], sl[wave][16 * n + c] = l[n];
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int i = 0; i < E / 4; ++i)
        *reinterpret_cast<f32x4*>(so + (wave * COLS + 16 * n + c) * PITCH + (4 * g + r) * E + 4 * i) =
            f32x4{o[n][4 * i][r], o[n][4 * i + 1][r], o[n][4 * i + 2][r], o[n][4 * i + 3][r]};
  }
  __syncthreads();
  // a column to 16 lanes
  if (G > 1 && wave >= 4) return;
#pragma unroll
  for (int n = 0; n < NC; ++n) {
    const int mine = 16 * n + (threadIdx.x >> 4), e0 = c * E, oc = c0 + mine, place = paOfGroup(a, min(oc, cols - 1)), h = kvh * group + (min(oc, cols - 1) - place * group);
    const int64_t row = s.start + s.first + place;
    float mAll = -INFINITY, sum = 0.f;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) mAll = fmaxf(mAll, sm[w][mine]);
    f32x4 v[E / 4] = {};
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
      const float weight = sm[w][mine] == -INFINITY ? 0.f : exp2f(sm[w][mine] - mAll);
      sum += sl[w][mine] * weight;
#pragma unroll
      for (int i = 0; i < E / 4; ++i)
#pragma unroll
        for (int k = 0; k < 4; ++k) v[i][k] += so[(w * COLS + mine) * PITCH + e0 + 4 * i + k] * weight;
    }
    bool odd = !(fabsf(sum) < INFINITY);
#pragma unroll
    for (int i = 0; i < E / 4; ++i)
#pragma unroll
      for (int k = 0; k < 4; ++k) odd |= !(fabsf(v[i][k]) < INFINITY);
    // columns whose sums are not finite: by themselves, with the tokens that they see alone
    const uint64_t bad = __builtin_amdgcn_ballot_w64(odd && oc < cols);
    if (oc < cols && (bad >> (lane & 48) & 0xffffu) == 0) {
      if (whole) {
        const float inv = sum == 0.f ? 0.f : 1.f / sum;
        float* out = reinterpret_cast<float*>(a.out) + row * a.oTok + (int64_t)h * a.oHead + e0;
#pragma unroll
        for (int i = 0; i < E / 4; ++i)
          if (!PART || e0 + 4 * i < a.d) *reinterpret_cast<f32x4*>(out + 4 * i) = v[i] * inv;
      } else {
        const int64_t slice = (ptPartialRow(x, s, b, place) * a.heads + h) * x.splits + split;
        if (c == 0) x.partialState[slice] = float2{mAll, sum};
#pragma unroll
        for (int i = 0; i < E / 4; ++i)
          if (!PART || e0 + 4 * i < a.d) *reinterpret_cast<f32x4*>(x.partial + slice * a.d + e0 + 4 * i) = v[i];
      }
    }
    for (int i = 0; i < 4; ++i)
      if ((bad >> (16 * i) & 0xffffu) != 0) pagedAgain<float, D>(x, s, b, kvh, locBase, span, t0, t1, split, whole, c0 + 16 * n + 4 * wave + i);
  }
}

template <int D, bool PART, int NC, int G>
__global__ __launch_bounds__(256 * G) void pagedFloatKernel(PtArgs x) {
  pagedPieces<kPtFloatCols * NC, 0>(x, [&](const PaSequence& s, int b, int kvh, int block, const PtSpan& span, int t0, int t1, int split, bool whole) {
    pagedFloatBlock<D, PART, NC, G>(x, s, b, kvh, block, span, t0, t1, split, whole);
  });
}

// Weights of `shares` partial results with (maximum, sum) `state` in lane i for share i: that share's in lane i, divided by the sum of all.
// *none: shares without a score, as bits. (shares <= 64)
__device__ __forceinline__ float pagedWeights(float2 state, int shares, uint64_t* none) {
  const int lane = threadIdx.x & 63;
  float m = lane < shares ? state.x : -INFINITY, l = lane < shares ? state.y : 0.f;
  const float most = waveMax(m);
  float w = m == -INFINITY ? 0.f : exp2f(m - most);
  if (l != l) w = l;  // (scores that are not numbers alone have no maximum)
  *none = __builtin_amdgcn_ballot_w64(w == 0.f && m == -INFINITY);
  const float sum = waveSum(l * w);
  return w * (sum == 0.f ? 0.f : 1.f / sum);
}

// The blocks of columns that were walked in shares: a wave joins MANY columns, four of them at a time with four shares of each on their way, or
// one with eight of them. Latency: 4 to 5 us.
template <typename T, int COLS, int FEW, int PAIRS, int MANY>
__global__ __launch_bounds__(256) void pagedMergeKernel(PtArgs x, int64_t step) {
  constexpr int kTogether = MANY == 1 ? 1 : 4, kBatch = MANY == 1 ? 8 : 4, kPtMergeCols = 4 * MANY;
  // d <= 128 PAIRS: a lane has elements 2 lane, 2 lane + 1 of every 128
  const PaArgs& a = x.a;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), kvh = blockIdx.x % a.kvHeads, group = a.group;
  for (int64_t u = blockIdx.x / a.kvHeads;; u += step) {
    const PaPlace at = paFind(a, u, [&](const PaSequence& s) {
      const int cols = ptColumns(a, s);
      return cols <= FEW ? 0 : (cols + kPtMergeCols - 1) / kPtMergeCols;
    });
    if (at.b < 0) return;
    const PaSequence& s = at.s;
    const int cols = ptColumns(a, s), origin = s.origin + s.first, first = at.at * kPtMergeCols + wave * (kPtMergeCols / 4);
#pragma unroll
    for (int c0 = 0; c0 < kPtMergeCols / 4; c0 += kTogether) {
      int shares[kTogether], most = 0;
      int64_t row[kTogether];
      int head[kTogether];
      float2 state[kTogether], acc[kTogether][PAIRS], v[kTogether][kBatch][PAIRS];
      const float* src[kTogether];
#pragma unroll
      for (int c = 0; c < kTogether; ++c) {
        const int col = min(first + c0 + c, cols - 1), place = paOfGroup(a, col), block = col / COLS;
        const PtSpan span(a, origin + paOfGroup(a, block * COLS), origin + paOfGroup(a, min(block * COLS + COLS - 1, cols - 1)));
        shares[c] = first + c0 + c < cols ? (span.tiles + x.tilesPerSplit - 1) / x.tilesPerSplit : 0;
        if (shares[c] <= 1) shares[c] = 0;  // (a block walked whole has its results)
        most = max(most, shares[c]);
        row[c] = s.start + s.first + place, head[c] = kvh * group + (col - place * group);
        const int64_t slice = (ptPartialRow(x, s, at.b, place) * a.heads + head[c]) * x.splits;
        state[c] = x.partialState[slice + min(lane, max(shares[c] - 1, 0))];
        src[c] = x.partial + slice * a.d;
#pragma unroll
        for (int k = 0; k < PAIRS; ++k) acc[c][k] = float2{0.f, 0.f};
      }
      uint64_t none[kTogether];
      float w[kTogether];
      for (int i0 = 0; i0 < most; i0 += kBatch) {
#pragma unroll
        for (int c = 0; c < kTogether; ++c)
#pragma unroll
          for (int i = 0; i < kBatch; ++i)
#pragma unroll
            for (int k = 0; k < PAIRS; ++k) {
              const int e = 2 * lane + 128 * k;
              v[c][i][k] = e < a.d && i0 + i < shares[c] ? *reinterpret_cast<const float2*>(src[c] + (i0 + i) * a.d + e) : float2{0.f, 0.f};
            }
#pragma unroll
        for (int c = 0; c < kTogether; ++c) {
          if (i0 == 0) w[c] = pagedWeights(state[c], shares[c], &none[c]);
#pragma unroll
          for (int i = 0; i < kBatch; ++i) {
            if (i0 + i >= shares[c] || (none[c] >> (i0 + i) & 1) != 0) continue;
            const float wi = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, w[c]), i0 + i));
#pragma unroll
            for (int k = 0; k < PAIRS; ++k) acc[c][k].x += wi * v[c][i][k].x, acc[c][k].y += wi * v[c][i][k].y;
          }
        }
      }
#pragma unroll
      for (int c = 0; c < kTogether; ++c) {
        if (shares[c] == 0) continue;
        T* out = reinterpret_cast<T*>(a.out) + row[c] * a.oTok + (int64_t)head[c] * a.oHead;
        typedef T Two __attribute__((ext_vector_type(2)));
#pragma unroll
        for (int k = 0; k < PAIRS; ++k) {
          const int e = 2 * lane + 128 * k;
          if (e < a.d) *reinterpret_cast<Two*>(out + e) = Two{static_cast<T>(acc[c][k].x), static_cast<T>(acc[c][k].y)};
        }
      }
    }
    if (u + step >= at.total) return;
  }
}

// The columns of sequences with few of them, `most` for each K/V head: a wave per column, or with WIDE a workgroup, whose waves take every
// fourth share. What does not depend on the lengths is asked for before they are there (shares without tokens were never written:
// what is read of them is left out). ROWS: partial results at the rows of q, which have to be found first (a variant, as what the others ask for
// would wait for that branch: 0.4 us).
template <typename T, bool WIDE, bool ROWS>
__global__ __launch_bounds__(256) void pagedFewMergeKernel(PtArgs x, int most) {
  constexpr int kPerLane = 4, kBatch = 8, kStep = WIDE ? 4 : 1;  // d <= 256
  __shared__ float red[WIDE ? 4 : 1][64 * kPerLane];
  const PaArgs& a = x.a;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), group = a.group;
  const int64_t i = WIDE ? (int64_t)blockIdx.x : (int64_t)blockIdx.x * 4 + wave, pair = i / most;
  const int col = (int)(i - pair * most), b = (int)(pair / a.kvHeads), kvh = (int)(pair - (int64_t)b * a.kvHeads);
  if (pair >= (int64_t)a.batch * a.kvHeads) return;
  int64_t slice = i;
  if constexpr (ROWS) {
    const PaSequence s = paSequence(a, b);
    if (col >= ptColumns(a, s)) return;
    slice = ptFewSlice(x, s, b, kvh, col);
  }
  const float* src = x.fewPartial + slice * x.fewSplits * (2 + a.d);
  const float2 state = *reinterpret_cast<const float2*>(src + min(lane, x.fewSplits - 1) * (2 + a.d));
  float v[kBatch][kPerLane], acc[kPerLane] = {0.f, 0.f, 0.f, 0.f};
  auto ask = [&](int first) {
#pragma unroll
    for (int k = 0; k < kBatch; ++k)
#pragma unroll
      for (int j = 0; j < kPerLane; ++j) {
        const int e = lane + 64 * j;
        v[k][j] = e < a.d ? src[min(first + kStep * k, x.fewSplits - 1) * (2 + a.d) + 2 + e] : 0.f;
      }
  };
  const int first = WIDE ? wave : 0;
  ask(first);
  const PaSequence s = paSequence(a, b);
  const int cols = ptColumns(a, s), shares = ptFewShares(x, s);
  if (col >= cols || cols > kPtFewCols || shares == 1) return;
  uint64_t none;
  const float w = pagedWeights(state, shares, &none);
  for (int i0 = first; i0 < shares; i0 += kStep * kBatch) {
    if (i0 != first) ask(i0);
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {
      const int share = i0 + kStep * k;
      if (share >= shares || (none >> share & 1) != 0) continue;
      const float wi = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, w), share));
#pragma unroll
      for (int j = 0; j < kPerLane; ++j) acc[j] += wi * v[k][j];
    }
  }
  const int place = paOfGroup(a, col);
  T* out = reinterpret_cast<T*>(a.out) + (s.start + s.first + place) * a.oTok + (int64_t)(kvh * group + (col - place * group)) * a.oHead;
  if (!WIDE) {
#pragma unroll
    for (int j = 0; j < kPerLane; ++j)
      if (lane + 64 * j < a.d) out[lane + 64 * j] = static_cast<T>(acc[j]);
    return;
  }
#pragma unroll
  for (int j = 0; j < kPerLane; ++j) red[wave][lane + 64 * j] = acc[j];
  __syncthreads();
  const int e = threadIdx.x;
  if (e < a.d) out[e] = static_cast<T>((red[0][e] + red[WIDE ? 1 : 0][e]) + (red[WIDE ? 2 : 0][e] + red[WIDE ? 3 : 0][e]));
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

template <typename T, int D>
static diopiError_t launchFew(hipStream_t stream, const PtArgs& x, int64_t pieces, bool wide) {
  constexpr int lds = kPfWaves * kPfStages * 2 * kPfTile * D * 2;
  static_assert(lds >= kPfWaves * 16 * (D + 4) * (int)sizeof(float) && lds <= 4 * kPtTile * D * 2, "the states have to fit in the ring, and the ring in the tiles");
  if (wide) {
    AMD_HIP(allowDynamicLds(reinterpret_cast<const void*>(&pagedFewKernel<T, D, true>), lds));
    hipLaunchKernelGGL((pagedFewKernel<T, D, true>), dim3((unsigned)(pieces * x.a.kvHeads / kPfWaves)), dim3(kPfWaves * 64), lds, stream, x);
  } else {
    AMD_HIP(allowDynamicLds(reinterpret_cast<const void*>(&pagedFewKernel<T, D, false>), lds));
    hipLaunchKernelGGL((pagedFewKernel<T, D, false>), dim3((unsigned)(pieces * x.a.kvHeads)), dim3(kPfWaves * 64), lds, stream, x);
  }
  AMD_LAUNCH_CHECK();
  return diopiSuccess;
}

template <int D, bool PART, int NC, int G>
static diopiError_t launchFloat(hipStream_t stream, const PtArgs& x, int64_t wgs) {
  constexpr int lds = 4 * G * kPtFloatCols * NC * (D + 4) * (int)sizeof(float);
  AMD_HIP(allowDynamicLds(reinterpret_cast<const void*>(&pagedFloatKernel<D, PART, NC, G>), lds));
  hipLaunchKernelGGL((pagedFloatKernel<D, PART, NC, G>), dim3((unsigned)wgs), dim3(256 * G), lds, stream, x);
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
  // columns of a sequence that paOfGroup divides (and 32 bits hold)
  const int64_t columns = std::min<int64_t>(a.maxNew, a.rows) * a.group + kPtCols;
  return columns < 1 << 30 && columns * a.group < (int64_t)1 << 32;
}

diopiError_t pagedAttentionMfma(diopiContextHandle_t ctx, hipStream_t stream, const PaArgs& a, diopiDtype_t dtype) {
  PtArgs x{};
  x.a = a;
  const bool wide = dtype == diopi_dtype_float32;
  if (!wide) x.kSlotBytes = (unsigned)(a.kSlotStride * 2), x.vSlotBytes = (unsigned)(a.vSlotStride * 2);
  const int64_t group = a.group, tokens = std::min<int64_t>(a.rows, (int64_t)a.batch * a.maxNew), cus = computeUnits();
  const int64_t tiles = std::max<int64_t>(1, std::min<int64_t>(ceilDiv(a.maxLen, kPtTile), ceilDiv(a.sinks, kPtTile) + ceilDiv((int64_t)a.window + kPtCols, kPtTile)));
  const int64_t limit = 1 << 24;  // workgroups: 2^32 threads
  const bool onlyFew = !wide && std::min<int64_t>(a.maxNew, a.rows) * group <= kPtFewCols;
  // Sequences of few columns, 16-bit rows: shares of at least 128 tokens, so many that two workgroups are there for each compute unit.
  bool wideHeads = false;
  const int64_t sequences = std::min<int64_t>(a.batch, tokens);
  const int64_t mostFew = kPtFewCols / group, fewTokens = std::min<int64_t>({mostFew, a.maxNew, a.rows});  // new tokens of a sequence of few columns
  if (!wide) {
    const int64_t seen = std::max<int64_t>(1, std::min<int64_t>(a.maxLen, (int64_t)a.sinks + a.window + kPtFewCols));
    const int64_t want = std::max<int64_t>(1, 2 * cus / (sequences * a.kvHeads));
    int64_t chunk = std::max<int64_t>({128, ceilDiv(ceilDiv(seen, want), 64) * 64, ceilDiv(ceilDiv(seen, kPtMaxSplit), 64) * 64});
    if (seen <= 256) chunk = seen;
    // next to blocks of columns, which take longer: shares of 4096, and no shares (nor a launch that joins them, 4.5 us) where the rows of q
    // are so many that no sequence has few, unless rows of none are among them (as in a recorded call for up to so many tokens: such a
    // sequence by itself takes 55 us for each 4096 of its cache, so only where new tokens are meant to be many)
    const int64_t others = (int64_t)(a.batch - 1) * a.maxNew;
    if (!onlyFew) chunk = a.maxNew >= kPtCols && a.rows - others > mostFew ? seen : std::max<int64_t>(chunk, std::min<int64_t>(seen, 4096));
    // A wave for each K/V head, with no shares, where a workgroup for each would be more than one round of them, of up to 128 tokens for each such
    // round and 512 (us, a workgroup -> a wave: 16 x 1 new token behind 130, 32 heads of 128, one round, 9.1 -> 15.3; 24 x 1 behind 60 12.8 -> 10.5, behind
    // 250 21.6 -> 22.1; 64 x 1, four rounds, behind 130 35.6 -> 27.0, behind 500 86.1 -> 83.3; 200 x 5, 32 heads on 8, behind 130 56.7 -> 30.7; 64 x 1
    // behind 1 ... 1000, lengths that differ much, 95 -> 111).
    const int64_t units = sequences * a.kvHeads, round = (a.d > 128 ? 1 : 2) * cus;
    wideHeads = onlyFew && a.kvHeads % kPfWaves == 0 && units > round && seen <= std::min<int64_t>(512, 128 * units / round);
    if (wideHeads) chunk = seen;
    if (fewTokens == 0) chunk = seen;  // (a token has more columns than that)
    x.fewChunk = (int)chunk, x.fewSplits = (int16_t)ceilDiv(seen, chunk);
    if (x.fewSplits > 1) {
      void* ws = nullptr;
      // Shares go by the sequences that have rows in q: of a batch with more sequences than that, partial results lie at the rows, which the launch that
      // joins them cannot find before it has the lengths.
      x.fewCols = a.batch <= tokens ? (int16_t)(fewTokens * group) : 0;
      const int64_t slices = x.fewCols != 0 ? (int64_t)a.batch * a.kvHeads * x.fewCols : a.rows * a.heads;
      AMD_TRY(requireWorkspace(ctx, slices * x.fewSplits * (2 + a.d) * (int64_t)sizeof(float), &ws));
      x.fewPartial = static_cast<float*>(ws);
    }
  }
  // The others: blocks of columns, what the rows of q fill, and one partly filled for each sequence but one at most. Where they leave compute
  // units without work the sequences are walked in shares.
  const int64_t columns = tokens * group;
  // fp32: two tiles of columns to a block where sequences have that many and there are blocks for half of the compute units all the same (us, one
  // tile -> two: 4 x 50 new tokens behind 100 ... 1000, 32 heads of 128 76 -> 61, 2 x 700 behind 300 361 -> 277; 16 x (1 .. 40), 8 heads of 64, 88
  // blocks, 11.5 -> 16.6). More than 128 elements leave no registers for it.
  const bool pairs = wide && a.d <= 128 && columns >= kPtFloatCols * sequences && ceilDiv(columns, 2 * kPtFloatCols) * a.kvHeads >= cus / 2;
  const int64_t blockCols = wide ? (pairs ? 2 : 1) * kPtFloatCols : kPtCols;
  const int64_t partly = std::max<int64_t>(1, wide ? sequences : std::min(sequences, columns / (kPtFewCols + 1))) - 1;
  const int64_t blocks = ceilDiv(columns, blockCols) + partly;
  x.tilesPerSplit = (int)tiles, x.splits = 1;
  if (!onlyFew) {
    // As many shares as make one round of workgroups, of at least 6 tiles, or two of 12 (fp32: 2, and three shares or none): partial results and
    // the launch that joins them cost a share of 6 tiles half as much again, and one workgroup alone on a compute unit takes 1.0 us for a tile
    // where each of two takes 2.3 (1 x 1024 new tokens, 32 heads, 16 tiles: 43 us in two shares, 33 in one). us, whole -> shares: 1 x 512 new tokens behind 8000, 32 heads on 8 218 -> 98, 1 x 300
    // behind 9000, 40 heads 220 -> 106, 1 x 64 behind 4000, 32 heads 105 -> 29, 4 x (200 .. 333) behind 100 ... 3000, 32 on 8 85 -> 68; against
    // it with more blocks than half a round: the same four next to 20 single tokens 92 -> 110, 4 x 512, 32 on 8 219 -> 254.
    const int64_t units = blocks * a.kvHeads, slots = (a.d > 128 ? 1 : 2) * cus, splits = (2 * slots + units) / (2 * units), least = wide ? 2 : 6;
    if (splits > (wide ? 2 : 1) && tiles >= (splits == 2 ? 4 : 2) * least) x.tilesPerSplit = (int)std::max<int64_t>({least, ceilDiv(tiles, splits), ceilDiv(tiles, kPtMaxSplit)});
    x.splits = (int)ceilDiv(tiles, x.tilesPerSplit);
    if (x.splits > 1) {
      void* ws = nullptr;
      const int64_t perSeq = std::min<int64_t>(a.maxNew, a.rows);
      if (a.batch * perSeq < a.rows) x.partialSeq = (int)perSeq;
      const int64_t slices = tokens * a.heads * x.splits;
      AMD_TRY(requireWorkspace(ctx, slices * (2 + a.d) * (int64_t)sizeof(float), &ws));
      x.partial = static_cast<float*>(ws), x.partialState = reinterpret_cast<float2*>(x.partial + slices * a.d);
    }
  }
  // fp32, a tile of columns to a block, no shares: eight waves, the tiles by turns to the first and the last four, where there are four tiles or more (us, four
  // waves -> eight: 16 x (1 .. 40) new tokens behind 0 .. 260, 8 heads of 64 12.2 -> 11.1, 8 x 1 behind 100 ... 1000, 32 heads of 128 46 -> 42; of two
  // tiles 8.4 -> 8.8, of shares of two 13.9 -> 16.4)
  const bool eight = wide && !pairs && (a.d == 64 || a.d == 128) && x.splits == 1 && tiles >= 4;  // (parts of a row: registers spill)
  const int64_t fewPieces = wide ? 0 : (int64_t)a.batch * x.fewSplits;
  x.tilePieces = onlyFew ? 0 : blocks * x.splits;
  const int64_t tileWgs = x.tilePieces * a.kvHeads, wgs = tileWgs + fewPieces * a.kvHeads;
  x.tileWgs = (unsigned)std::min(tileWgs, limit);
  x.turn = tileWgs <= 2 * cus ? ceilDiv(cus, a.kvHeads) : x.tilePieces;
  AMD_CHECK(wgs < limit, "paged attention: %ld rows of %d heads exceed the grid limits", (long)a.rows, a.heads);
#define SIZE_CALL(CALL)               \
  do {                                \
    if (a.d <= 64) CALL(64);          \
    else if (a.d <= 128) CALL(128);   \
    else CALL(256);                   \
  } while (0)
#define HALF_CALL(T, D) AMD_TRY((onlyFew ? launchFew<T, D>(stream, x, fewPieces, wideHeads) : a.d == D ? launchTile<T, D, false>(stream, x, wgs) : launchTile<T, D, true>(stream, x, wgs)))
#define BF16_CALL(D) HALF_CALL(bf16_t, D)
#define FP16_CALL(D) HALF_CALL(half_t, D)
#define FP32_CALL_AS(D, NC) AMD_TRY((a.d == D ? launchFloat<D, false, NC, 1>(stream, x, wgs) : launchFloat<D, true, NC, 1>(stream, x, wgs)))
#define FP32_CALL(D)                                       \
  do {                                                     \
    if constexpr (D <= 128) {                              \
      if (pairs) FP32_CALL_AS(D, 2);                       \
      else if (eight) AMD_TRY((launchFloat<D, false, 1, 2>(stream, x, wgs))); \
      else FP32_CALL_AS(D, 1);                             \
    } else {                                               \
      FP32_CALL_AS(D, 1);                                  \
    }                                                      \
  } while (0)
  if (dtype == diopi_dtype_bfloat16) SIZE_CALL(BF16_CALL);
  else if (dtype == diopi_dtype_float16) SIZE_CALL(FP16_CALL);
  else SIZE_CALL(FP32_CALL);
#undef FP32_CALL
#undef FP32_CALL_AS
#undef FP16_CALL
#undef BF16_CALL
#undef HALF_CALL
#undef SIZE_CALL
  if (x.fewSplits > 1) {
    const int mostCols = (int)(fewTokens * group);
    const bool wideMerge = x.fewSplits > 8;
    const int64_t merges = ceilDiv((int64_t)a.batch * a.kvHeads * mostCols, wideMerge ? 1 : 4);
    AMD_CHECK(merges < limit, "paged attention: %d sequences of %d heads exceed the grid limits", a.batch, a.heads);
#define FEW_MERGE_AS(T, WIDE, ROWS) hipLaunchKernelGGL((pagedFewMergeKernel<T, WIDE, ROWS>), dim3((unsigned)merges), dim3(256), 0, stream, x, mostCols)
#define FEW_MERGE(T)                                      \
  do {                                                    \
    if (wideMerge && x.fewCols == 0) FEW_MERGE_AS(T, true, true); \
    else if (wideMerge) FEW_MERGE_AS(T, true, false);     \
    else if (x.fewCols == 0) FEW_MERGE_AS(T, false, true); \
    else FEW_MERGE_AS(T, false, false);                   \
  } while (0)
    if (dtype == diopi_dtype_bfloat16) FEW_MERGE(bf16_t);
    else FEW_MERGE(half_t);
#undef FEW_MERGE
#undef FEW_MERGE_AS
    AMD_LAUNCH_CHECK();
  }
  if (x.splits > 1) {
    // a wave per column where that is less than four workgroups for a compute unit
    const bool single = columns * a.kvHeads < 16 * cus;
    const int64_t pieces = ceilDiv(columns, single ? 4 : 32) + partly;
    AMD_CHECK(pieces * a.kvHeads < limit, "paged attention: %ld rows of %d heads exceed the grid limits", (long)a.rows, a.heads);
    const dim3 grid((unsigned)(pieces * a.kvHeads)), block(256);
#define TILE_MERGE(T, COLS, FEW)                                                                                                        \
  do {                                                                                                                                  \
    if (single && a.d <= 128) hipLaunchKernelGGL((pagedMergeKernel<T, COLS, FEW, 1, 1>), grid, block, 0, stream, x, pieces);             \
    else if (single) hipLaunchKernelGGL((pagedMergeKernel<T, COLS, FEW, 2, 1>), grid, block, 0, stream, x, pieces);                      \
    else if (a.d <= 128) hipLaunchKernelGGL((pagedMergeKernel<T, COLS, FEW, 1, 8>), grid, block, 0, stream, x, pieces);                  \
    else hipLaunchKernelGGL((pagedMergeKernel<T, COLS, FEW, 2, 8>), grid, block, 0, stream, x, pieces);                                  \
  } while (0)
    if (dtype == diopi_dtype_bfloat16) TILE_MERGE(bf16_t, kPtCols, kPtFewCols);
    else if (dtype == diopi_dtype_float16) TILE_MERGE(half_t, kPtCols, kPtFewCols);
    else if (pairs) TILE_MERGE(float, 2 * kPtFloatCols, 0);
    else TILE_MERGE(float, kPtFloatCols, 0);
#undef TILE_MERGE
    AMD_LAUNCH_CHECK();
  }
  return diopiSuccess;
}

}  // namespace amd
