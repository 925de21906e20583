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
};

// Any head size up to 1024: one workgroup per (sequence, head) walks the shared tokens and then its own, 256 at a time, one
// token's dot product per thread and P.V with the threads over d. A correctness path.
template <typename T>
__global__ __launch_bounds__(256) void decodePrefixAnyKernel(TaPrefixArgs x, T* __restrict__ out) {
  __shared__ float prob[256];
  __shared__ int64_t slotOf[256];
  __shared__ float red[4];
  const TaArgs& a = x.a;
  const int h = blockIdx.x, b = blockIdx.y, tid = threadIdx.x;
  const int len = (int)min(max(ldIndex(a.bLen, b, a.len64), (int64_t)0), (int64_t)a.maxLen), all = x.len + len;
  const int kvh = h / (a.heads / a.kvHeads);
  const int64_t locBase = (int64_t)b * a.locRowStride + (a.maxLen - len);
  const T* q = reinterpret_cast<const T*>(a.q) + b * a.qBatchStride + h * a.qHeadStride;
  const T* kHead = reinterpret_cast<const T*>(a.k) + kvh * a.kHeadStride;
  const T* vHead = reinterpret_cast<const T*>(a.v) + kvh * a.vHeadStride;
  float m = -INFINITY, l = 0.f, acc[4] = {0.f, 0.f, 0.f, 0.f};  // acc[j]: element tid + 256 j of the output row
  for (int t0 = 0; t0 < all; t0 += 256) {
    const int t = t0 + tid;
    int64_t slot = t >= all ? -1 : t < x.len ? ldIndex(x.loc, t, x.loc64) : ldIndex(a.bLoc, locBase + (t - x.len), a.loc64);
    if (slot >= a.slots) slot = -1;
    float sc = -INFINITY;  // in units of log2
    if (slot >= 0) {
      const T* k = kHead + slot * a.kSlotStride;
      float d = 0.f;
      for (int e = 0; e < a.d; ++e) d += static_cast<float>(q[e]) * static_cast<float>(k[e]);
      sc = d * a.scaleLog2e;
    }
    const float mn = fmaxf(m, blockMax256(sc, red));
    const float ref = mn == -INFINITY ? 0.f : mn;
    const float pr = slot < 0 ? 0.f : exp2f(sc - ref);
    prob[tid] = pr;
    slotOf[tid] = slot;
    const float bs = blockSum256(pr, red);  // its barriers also publish prob / slotOf
    const float corr = m == -INFINITY ? 1.f : exp2f(m - ref);  // (no maximum yet: the sums are 0, or NaN)
    l = l * corr + bs;
    const int cnt = min(256, all - t0);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int e = tid + 256 * j;
      if (e < a.d) {
        float o = acc[j] * corr;
        for (int i = 0; i < cnt; ++i)
          if (slotOf[i] >= 0) o += prob[i] * static_cast<float>(vHead[slotOf[i] * a.vSlotStride + e]);
        acc[j] = o;
      }
    }
    m = mn;
    __syncthreads();  // prob / slotOf are rewritten by the next block of tokens
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int e = tid + 256 * j;
    if (e < a.d) out[((int64_t)b * a.heads + h) * a.d + e] = static_cast<T>(acc[j] * inv);
  }
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
  AMD_CHECK(prefix.shape[0] + (int64_t)maxInputLen < ((int64_t)1 << 31) - 256, "shared prefix attention: %ld shared tokens and %d own ones exceed 2^31",
            (long)prefix.shape[0], maxInputLen);
  AMD_CHECK(out.defined() && out.dtype == t.q.dtype && out.ndim == 3 && out.isContiguous(), "shared prefix attention: out must be a dense tensor shaped like q");
  for (int d = 0; d < 3; ++d) AMD_CHECK(out.shape[d] == t.q.shape[d], "shared prefix attention: out must be shaped like q");
  if (t.q.numel == 0) return diopiSuccess;
  AMD_CHECK(a.batch <= 65535, "shared prefix attention: batch %d exceeds the grid limits", a.batch);
  AMD_CHECK(t.q.shape[2] <= kTaGenericMaxD, "shared prefix attention: head_dim %ld exceeds %d", (long)t.q.shape[2], kTaGenericMaxD);
  AMD_TRY(makeContiguous(ctx, stream, prefix, &densePrefix));
  x.loc = densePrefix.data, x.loc64 = prefix.dtype == diopi_dtype_int64, x.len = (int)prefix.shape[0];
  const dim3 grid(a.heads, a.batch);
  if (t.q.dtype == diopi_dtype_bfloat16) hipLaunchKernelGGL((decodePrefixAnyKernel<bf16_t>), grid, dim3(256), 0, stream, x, out.ptr<bf16_t>());
  else if (t.q.dtype == diopi_dtype_float16) hipLaunchKernelGGL((decodePrefixAnyKernel<half_t>), grid, dim3(256), 0, stream, x, out.ptr<half_t>());
  else hipLaunchKernelGGL((decodePrefixAnyKernel<float>), grid, dim3(256), 0, stream, x, out.ptr<float>());
  AMD_LAUNCH_CHECK();
  return diopiSuccess;
}
