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
};

// Any head size up to 1024: one workgroup per (sequence, head), 256 tokens at a time, one token's dot product per thread and
// P.V with the threads over d. A correctness path.
template <typename T>
__global__ __launch_bounds__(256) void decodeInt8AnyKernel(TaInt8Args x, T* __restrict__ out) {
  __shared__ float prob[256];
  __shared__ int64_t slotOf[256];
  __shared__ float red[4];
  const TaArgs& a = x.a;
  const int h = blockIdx.x, b = blockIdx.y, tid = threadIdx.x;
  const int len = (int)min(max(ldIndex(a.bLen, b, a.len64), (int64_t)0), (int64_t)a.maxLen);
  const int kvh = h / (a.heads / a.kvHeads);
  const int64_t locBase = (int64_t)b * a.locRowStride + (a.maxLen - len);
  const T* q = reinterpret_cast<const T*>(a.q) + b * a.qBatchStride + h * a.qHeadStride;
  const int8_t* kHead = reinterpret_cast<const int8_t*>(a.k) + kvh * a.kHeadStride;
  const int8_t* vHead = reinterpret_cast<const int8_t*>(a.v) + kvh * a.vHeadStride;
  float m = -INFINITY, l = 0.f, acc[4] = {0.f, 0.f, 0.f, 0.f};  // acc[j]: element tid + 256 j of the output row
  for (int t0 = 0; t0 < len; t0 += 256) {
    const int t = t0 + tid;
    int64_t slot = t < len ? ldIndex(a.bLoc, locBase + t, a.loc64) : -1;
    if (slot >= a.slots) slot = -1;
    float sc = -INFINITY, vs = 0.f;  // the score in units of log2; the scale of V
    if (slot >= 0) {
      const int8_t* k = kHead + slot * a.kSlotStride;
      float d = 0.f;
      for (int e = 0; e < a.d; ++e) d += static_cast<float>(q[e]) * static_cast<float>(k[e]);
      sc = d * (x.kScale[slot * x.kScaleSlot + kvh * x.kScaleHead] * a.scaleLog2e);
      vs = x.vScale[slot * x.vScaleSlot + kvh * x.vScaleHead];
    }
    const float mn = fmaxf(m, blockMax256(sc, red));
    const float ref = mn == -INFINITY ? 0.f : mn;  // (scores that are NaN leave no maximum, and make all of the row NaN)
    const float pr = slot < 0 ? 0.f : exp2f(sc - ref);
    prob[tid] = pr * vs;
    slotOf[tid] = slot;
    const float bs = blockSum256(pr, red);  // its barriers also publish prob / slotOf
    const float corr = m == -INFINITY ? 1.f : exp2f(m - ref);  // (no maximum yet: the sums are 0, or NaN)
    l = l * corr + bs;
    const int cnt = min(256, len - t0);
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
  const dim3 grid(a.heads, a.batch);
  if (t.q.dtype == diopi_dtype_bfloat16) hipLaunchKernelGGL((decodeInt8AnyKernel<bf16_t>), grid, dim3(256), 0, stream, x, out.ptr<bf16_t>());
  else if (t.q.dtype == diopi_dtype_float16) hipLaunchKernelGGL((decodeInt8AnyKernel<half_t>), grid, dim3(256), 0, stream, x, out.ptr<half_t>());
  else hipLaunchKernelGGL((decodeInt8AnyKernel<float>), grid, dim3(256), 0, stream, x, out.ptr<float>());
  AMD_LAUNCH_CHECK();
  return diopiSuccess;
}
