// Decode attention over rows of any size and layout, of a pool of q's type or an int8 one (see token_attention_int8.hip), behind shared
// tokens or not (token_attention_prefix.hip), for gfx950. Bound by the vector ALUs: a row serves one query head, its dot product is a
// sum over the wave's lanes. Rows that the matrix pipe does not take, us, with a dot product to a
// thread and a workgroup to a (sequence, head) -> this: int8, 4 x 3000 tokens, 8 heads of 100 1033 -> 33, 32 x (50 .. 500), 32 on 8 280 -> 70, 8 x
// (500 .. 1000), 8 heads of 320 on 2, fp32 707 -> 174; own tokens of fp32 heads of 256, 2 x (177 .. 621), 64 on 8, behind 6237 shared
// ones, all of it 2794 -> 71; 3000 shared, 32 x (50 .. 500), 32 heads of 100 on 8, bf16, which share nothing here, 367.
#include <algorithm>
#include <type_traits>

#include "token_attention.hpp"

namespace amd {

// Any head size up to 64 J, any strides: a workgroup per (sequence, head, chunk) walks the first x.walked shared tokens and the
// sequence's own, a wave a token at a time with the row spread over its lanes (K and V in whole lines), UNR of them asked for
// at once; slots are looked up 64 at a time. The one of several chunks that is not the first and has no tokens writes nothing.
constexpr int kPaWaves = 4;
template <typename T, bool INT8, int J, int UNR>
__global__ __launch_bounds__(kPaWaves * 64) void decodeAnyKernel(TaAnyArgs x, T* __restrict__ out, float* __restrict__ partial) {
  using P = std::conditional_t<INT8, int8_t, T>;
  __shared__ float red[kPaWaves][64 * J], state[kPaWaves][2];
  const TaArgs& a = x.a;
  const int h = blockIdx.x, b = blockIdx.y, split = blockIdx.z, lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int len = cutLength(a.bLen, b, a.len64, a.maxLen), all = x.walked + len;
  const int begin = split * x.chunk, end = min(all, begin + x.chunk);
  if (begin >= all && split != 0) return;
  const int kvh = h / (a.heads / a.kvHeads);
  const int64_t locBase = (int64_t)b * a.locRowStride + (a.maxLen - len);
  const T* q = reinterpret_cast<const T*>(a.q) + b * a.qBatchStride + h * a.qHeadStride;
  const P* kHead = reinterpret_cast<const P*>(a.k) + kvh * a.kHeadStride;
  const P* vHead = reinterpret_cast<const P*>(a.v) + kvh * a.vHeadStride;
  int at[J];  // the lane's elements of a row; past its end the first one, which q's zero leaves out
  float qf[J], acc[J], m = -INFINITY, l = 0.f;
#pragma unroll
  for (int j = 0; j < J; ++j) {
    const int e = lane + 64 * j;
    at[j] = e < a.d ? e : 0;
    qf[j] = e < a.d ? static_cast<float>(q[e]) * a.scaleLog2e : 0.f;
    acc[j] = 0.f;
  }
  for (int t0 = begin + wave * 64; t0 < end; t0 += kPaWaves * 64) {
    const int t = min(t0 + lane, end - 1), cnt = min(64, end - t0);
    int64_t mine = t < x.walked ? ldIndex(x.loc, t, x.locIs64) : ldIndex(a.bLoc, locBase + (t - x.walked), a.loc64);
    if (mine < 0 || mine >= a.slots) mine = -1;  // slots outside the pool are skipped, never dereferenced
    for (int i = 0; i < cnt; i += UNR) {
      float k[UNR][J], v[UNR][J], ks[UNR], vs[UNR], sc[UNR], mt = m;
      bool counts[UNR];
#pragma unroll
      for (int u = 0; u < UNR; ++u) {
        const int from = min(i + u, cnt - 1);
        const int64_t slot = (int64_t)((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(mine >> 32), from) << 32 | (uint32_t)__builtin_amdgcn_readlane((int)mine, from));
        counts[u] = i + u < cnt && slot >= 0;
        const P* kRow = kHead + max(slot, (int64_t)0) * a.kSlotStride;
        const P* vRow = vHead + max(slot, (int64_t)0) * a.vSlotStride;
#pragma unroll
        for (int j = 0; j < J; ++j) k[u][j] = static_cast<float>(kRow[at[j]]), v[u][j] = static_cast<float>(vRow[at[j]]);
        ks[u] = INT8 ? x.kScale[max(slot, (int64_t)0) * x.kScaleSlot + kvh * x.kScaleHead] : 1.f;
        vs[u] = INT8 ? x.vScale[max(slot, (int64_t)0) * x.vScaleSlot + kvh * x.vScaleHead] : 1.f;
      }
#pragma unroll
      for (int u = 0; u < UNR; ++u) {
        float d = 0.f;
#pragma unroll
        for (int j = 0; j < J; ++j) d += lane + 64 * j < a.d ? qf[j] * k[u][j] : 0.f;
        sc[u] = waveSum(d) * ks[u];
        if (!counts[u]) sc[u] = -INFINITY;
        mt = fmaxf(mt, sc[u]);
      }
      const float ref = mt == -INFINITY ? 0.f : mt, corr = m == -INFINITY ? 1.f : exp2f(m - ref);  // (no maximum yet: the sums are 0, or NaN)
      m = mt, l *= corr;
#pragma unroll
      for (int j = 0; j < J; ++j) acc[j] *= corr;
#pragma unroll
      for (int u = 0; u < UNR; ++u) {
        if (!counts[u]) continue;
        const float p = exp2f(behindRounded(sc[u], ref));
        l += p;
        const float w = p * vs[u];
#pragma unroll
        for (int j = 0; j < J; ++j) acc[j] += w * v[u][j];
      }
    }
  }
  if (l != l && m == -INFINITY) m = 0.f;  // scores that are not numbers alone: as a maximum of minus infinity they would be left out
  if (lane == 0) state[wave][0] = m, state[wave][1] = l;
#pragma unroll
  for (int j = 0; j < J; ++j) red[wave][lane + 64 * j] = acc[j];
  __syncthreads();
  float mAll = -INFINITY, lAll = 0.f, w[kPaWaves];
#pragma unroll
  for (int i = 0; i < kPaWaves; ++i) mAll = fmaxf(mAll, state[i][0]);
#pragma unroll
  for (int i = 0; i < kPaWaves; ++i) {
    w[i] = state[i][0] == -INFINITY ? 0.f : exp2f(state[i][0] - mAll);
    lAll += state[i][1] * w[i];
  }
  const int64_t pair = (int64_t)b * a.heads + h;
  float* const dst = partial + (pair * x.split + split) * (2 + a.d);
  if (partial != nullptr && threadIdx.x == 0) dst[0] = mAll, dst[1] = lAll;
  const float inv = lAll == 0.f ? 0.f : 1.f / lAll;
  for (int e = threadIdx.x; e < a.d; e += kPaWaves * 64) {
    float o = 0.f;
#pragma unroll
    for (int i = 0; i < kPaWaves; ++i) o += red[i][e] * w[i];
    if (partial != nullptr) dst[2 + e] = o;
    else out[pair * a.d + e] = static_cast<T>(o * inv);
  }
}

// Four workgroups to a compute unit, chunks of whole rounds of the waves.
diopiError_t walkAny(diopiContextHandle_t ctx, hipStream_t stream, TaAnyArgs x, diopiDtype_t dtype, void* out, bool alone, TaPartials* own) {
  const TaArgs& a = x.a;
  const int64_t pairs = (int64_t)a.batch * a.heads, total = std::max<int64_t>(1, (int64_t)x.walked + a.maxLen);
  const int64_t most = std::min<int64_t>(kTaMaxSplit, std::max<int64_t>(1, 4 * computeUnits() / pairs));
  x.chunk = (int)(ceilDiv(ceilDiv(total, most), kPaWaves * 64) * kPaWaves * 64);
  x.split = (int)ceilDiv(total, x.chunk);
  AMD_CHECK(pairs < 1 << 24, "token attention: %d sequences of %d heads exceed the grid limits", a.batch, a.heads);  // (2^32 threads)
  float* partial = nullptr;
  if (!alone || x.split > 1) {
    void* ws = nullptr;
    AMD_TRY(requireWorkspace(ctx, pairs * x.split * (2 + a.d) * (int64_t)sizeof(float), &ws));
    partial = static_cast<float*>(ws);
  }
  const dim3 grid(a.heads, a.batch, x.split);
#define ANY_CALL_SIZE(T, J, UNR)                                                                                                                              \
  do {                                                                                                                                                        \
    if (x.kScale != nullptr) hipLaunchKernelGGL((decodeAnyKernel<T, true, J, UNR>), grid, dim3(kPaWaves * 64), 0, stream, x, static_cast<T*>(out), partial);     \
    else hipLaunchKernelGGL((decodeAnyKernel<T, false, J, UNR>), grid, dim3(kPaWaves * 64), 0, stream, x, static_cast<T*>(out), partial);                        \
  } while (0)
#define ANY_CALL(T)                                       \
  do {                                                    \
    if (a.d <= 64) ANY_CALL_SIZE(T, 1, 8);                \
    else if (a.d <= 128) ANY_CALL_SIZE(T, 2, 8);          \
    else if (a.d <= 256) ANY_CALL_SIZE(T, 4, 4);          \
    else ANY_CALL_SIZE(T, kTaGenericMaxD / 64, 1);        \
  } while (0)
  if (dtype == diopi_dtype_bfloat16) ANY_CALL(bf16_t);
  else if (dtype == diopi_dtype_float16) ANY_CALL(half_t);
  else ANY_CALL(float);
#undef ANY_CALL
#undef ANY_CALL_SIZE
  AMD_LAUNCH_CHECK();
  *own = TaPartials{partial, partial ? x.split : 0, x.chunk, 0.f};
  return diopiSuccess;
}

}  // namespace amd
