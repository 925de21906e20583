// Attention of the new tokens of each sequence over all that a paged pool holds of it, for gfx950.
//
//   q [rows, heads, d]             rows b_start_loc[b] ... + b_new_len[b] are the new tokens of sequence b
//   k, v [slots, kv_heads, d]      the pool; the new tokens are in it already
//   b_loc [batch, >= max_len]      slot table, right-aligned: token j of sequence b is at column max_len - seq_len[b] + j
//
// New token t stands at position p = seq_len[b] - new_len[b] + t and sees the tokens j <= p, with a window of W only the W
// last of those and the first S of the sequence (j > p - W or j < S):
//   out = softmax_j(q . k[slot_j] / sqrt(d)) . v[slot_j]
// Scores, softmax and sums are in fp32. A piece of a prompt, speculated tokens and decoding sequences are the same thing here;
// the reference knows the two ends alone, prompts without a cache and single tokens (dicp/dicp/vendor/AscendGraph/ext_ops.py:52-133).
//
// This file holds the entry points and the kernel for rows of any kind.
#include <algorithm>
#include <type_traits>

#include "paged_attention.hpp"

namespace amd {

// Any head size up to 64 J, any strides: a workgroup per (new token, head), whose waves take 64 tokens that it sees in turn (PaColumn).
// Bound by the vector ALUs, whose sums over the lanes cost more than the products. Rows one element off 16-byte pieces, against aligned ones on the matrix
// pipe: 4 x 128 new tokens behind 1000, 32 heads of 128 on 8, bf16 1.5 ms, 39 us; 48 single tokens with a window of 2048, the same heads in fp16 376 us, 72 us.
constexpr int kPgWaves = 4;
template <typename T, int J, int UNR>
__global__ __launch_bounds__(kPgWaves * 64) void pagedAnyKernel(PaArgs a) {
  __shared__ float red[kPgWaves][64 * J], state[kPgWaves][2];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int h = blockIdx.x % a.heads, kvh = h / (a.heads / a.kvHeads);
  for (int64_t u = blockIdx.x / a.heads;; u += gridDim.x / a.heads) {
    const PaPlace at = paFind(a, u, [](const PaSequence& s) { return s.end - s.first; });
    if (at.b < 0) return;
    const PaSequence& s = at.s;
    const int t = s.first + at.at, p = s.origin + t;
    const int64_t row = s.start + t;
    const int64_t locBase = (int64_t)at.b * a.locRowStride + (a.maxLen - s.len);
    int head, low;
    paSeen(a, p, &head, &low);
    PaColumn<T, J, UNR> c;
    c.walk(a, reinterpret_cast<const T*>(a.q) + row * a.qTok + h * a.qHead, kvh, locBase, 0, head, low, p + 1, wave * 64, kPgWaves * 64);
    __syncthreads();  // (the sums of the token before have been read)
    if (lane == 0) state[wave][0] = c.m, state[wave][1] = c.l;
#pragma unroll
    for (int j = 0; j < J; ++j) red[wave][lane + 64 * j] = c.acc[j];
    __syncthreads();
    float mAll = -INFINITY, lAll = 0.f, w[kPgWaves];
#pragma unroll
    for (int i = 0; i < kPgWaves; ++i) mAll = fmaxf(mAll, state[i][0]);
#pragma unroll
    for (int i = 0; i < kPgWaves; ++i) {
      w[i] = state[i][0] == -INFINITY ? 0.f : exp2f(state[i][0] - mAll);
      lAll += state[i][1] * w[i];
    }
    const float inv = lAll == 0.f ? 0.f : 1.f / lAll;
    T* out = reinterpret_cast<T*>(a.out) + row * a.oTok + h * a.oHead;
    for (int e = threadIdx.x; e < a.d; e += kPgWaves * 64) {
      float o = 0.f;
#pragma unroll
      for (int i = 0; i < kPgWaves; ++i) o += red[i][e] * w[i];
      out[e] = static_cast<T>(o * inv);
    }
    if (u + gridDim.x / a.heads >= at.total) return;
  }
}

diopiError_t pagedAttentionAny(hipStream_t stream, const PaArgs& a, diopiDtype_t dtype) {
  const int64_t wgs = a.rows * a.heads;  // (sequences that share rows of q are more pieces: the workgroups take several)
  AMD_CHECK(wgs < 1 << 24, "paged attention: %ld rows of %d heads exceed the grid limits", (long)a.rows, a.heads);  // (2^32 threads)
#define ANY_CALL_SIZE(T, J, UNR) hipLaunchKernelGGL((pagedAnyKernel<T, J, UNR>), dim3((unsigned)wgs), dim3(kPgWaves * 64), 0, stream, a)
#define ANY_CALL(T)                                \
  do {                                             \
    if (a.d <= 64) ANY_CALL_SIZE(T, 1, 8);         \
    else if (a.d <= 128) ANY_CALL_SIZE(T, 2, 8);   \
    else if (a.d <= 256) ANY_CALL_SIZE(T, 4, 4);   \
    else ANY_CALL_SIZE(T, kTaGenericMaxD / 64, 1); \
  } while (0)
  if (dtype == diopi_dtype_bfloat16) ANY_CALL(bf16_t);
  else if (dtype == diopi_dtype_float16) ANY_CALL(half_t);
  else ANY_CALL(float);
#undef ANY_CALL
#undef ANY_CALL_SIZE
  AMD_LAUNCH_CHECK();
  return diopiSuccess;
}

static diopiError_t checkWindow(int window, int sinks, int maxLen, PaArgs* a) {
  AMD_CHECK(window >= 0 && sinks >= 0, "paged attention: a window of %d tokens and %d first ones", window, sinks);
  AMD_CHECK(maxLen <= 1 << 30, "paged attention: sequences of %d tokens exceed 2^30", maxLen);
  a->window = window == 0 ? maxLen : std::min(window, std::max(maxLen, 1));
  a->sinks = std::min(sinks, maxLen);
  return diopiSuccess;
}

static diopiError_t checkLengths(const TensorView& t, int64_t batch, const char* name) {
  AMD_CHECK(t.defined(), "paged attention: %s is null", name);
  AMD_CHECK(t.dtype == diopi_dtype_int32 || t.dtype == diopi_dtype_int64, "paged attention: %s must be int32 or int64, got %s", name, dtypeName(t.dtype));
  AMD_CHECK(t.numel == batch && t.isContiguous(), "paged attention: %s must be dense with %ld entries", name, (long)batch);
  return diopiSuccess;
}

}  // namespace amd

using namespace amd;

extern "C" __attribute__((visibility("default"))) diopiError_t diopiPagedContextAttentionInference(
    diopiContextHandle_t ctx, diopiTensorHandle_t outH, diopiConstTensorHandle_t qH, diopiConstTensorHandle_t kH,
    diopiConstTensorHandle_t vH, diopiConstTensorHandle_t locH, diopiConstTensorHandle_t startH, diopiConstTensorHandle_t newH,
    diopiConstTensorHandle_t lenH, int maxNewLen, int maxInputLen, int window, int sinks) {
  hipStream_t stream;
  AMD_TRY(getStream(ctx, &stream));
  TensorView out, q, k, v, loc, start, fresh, len;
  AMD_TRY(getView(outH, &out, "out"));
  AMD_TRY(getView(qH, &q, "q"));
  AMD_TRY(getView(kH, &k, "k"));
  AMD_TRY(getView(vH, &v, "v"));
  AMD_TRY(getView(locH, &loc, "b_loc"));
  AMD_TRY(getView(startH, &start, "b_start_loc"));
  AMD_TRY(getView(newH, &fresh, "b_new_len"));
  AMD_TRY(getView(lenH, &len, "b_seq_len"));
  AMD_CHECK(q.defined() && q.ndim == 3, "paged attention: q must be [tokens, heads, head_dim]");
  AMD_CHECK(q.dtype == diopi_dtype_bfloat16 || q.dtype == diopi_dtype_float16 || q.dtype == diopi_dtype_float32, "paged attention: unsupported dtype %s",
            dtypeName(q.dtype));
  AMD_CHECK(out.defined() && out.ndim == 3 && out.dtype == q.dtype, "paged attention: out must have q's shape and dtype");
  AMD_CHECK(k.defined() && k.ndim == 3 && v.defined() && v.ndim == 3, "paged attention: k and v must be [slots, kv_heads, head_dim]");
  AMD_CHECK(k.dtype == q.dtype && v.dtype == q.dtype, "paged attention: k and v are %s and %s, q is %s", dtypeName(k.dtype), dtypeName(v.dtype), dtypeName(q.dtype));
  for (int d = 0; d < 3; ++d) {
    AMD_CHECK(out.shape[d] == q.shape[d], "paged attention: out must have q's shape and dtype");
    AMD_CHECK(k.shape[d] == v.shape[d], "paged attention: k and v differ at dim %d", d);
  }
  AMD_CHECK(k.shape[2] == q.shape[2], "paged attention: head_dim mismatch (%ld and %ld)", (long)k.shape[2], (long)q.shape[2]);
  AMD_CHECK(q.shape[2] <= kTaGenericMaxD, "paged attention: head_dim %ld exceeds %d", (long)q.shape[2], kTaGenericMaxD);
  AMD_CHECK(k.shape[1] > 0 && q.shape[1] % k.shape[1] == 0, "paged attention: %ld heads are not a multiple of %ld kv heads", (long)q.shape[1], (long)k.shape[1]);
  auto unit = [](const TensorView& t) { return t.stride[2] == 1 || t.shape[2] == 1; };
  AMD_CHECK(unit(q) && unit(k) && unit(v) && unit(out), "paged attention: head_dim of q, k, v and out must be contiguous");
  AMD_CHECK(k.shape[0] > 0, "paged attention: the KV pool has no slots");
  AMD_CHECK(loc.defined() && loc.ndim == 2 && (loc.dtype == diopi_dtype_int32 || loc.dtype == diopi_dtype_int64) && (loc.stride[1] == 1 || loc.shape[1] <= 1),
            "paged attention: b_loc must be [batch, n] of int32 or int64 with a contiguous last dim");
  const int64_t batch = loc.shape[0];
  AMD_TRY(checkLengths(start, batch, "b_start_loc"));
  AMD_TRY(checkLengths(fresh, batch, "b_new_len"));
  AMD_TRY(checkLengths(len, batch, "b_seq_len"));
  AMD_CHECK(maxNewLen >= 0 && maxInputLen >= 0 && loc.shape[1] >= maxInputLen, "paged attention: b_loc has %ld columns, max_new_len is %d and max_input_len %d",
            (long)loc.shape[1], maxNewLen, maxInputLen);
  PaArgs a{};
  AMD_TRY(checkWindow(window, sinks, maxInputLen, &a));
  AMD_CHECK(batch <= 65535, "paged attention: batch %ld exceeds the grid limits", (long)batch);
  if (batch == 0 || q.numel == 0 || maxNewLen == 0) return diopiSuccess;
  a.q = q.data, a.k = k.data, a.v = v.data, a.out = out.data;
  a.bLoc = loc.data, a.bStart = start.data, a.bNew = fresh.data, a.bLen = len.data;
  a.loc64 = loc.dtype == diopi_dtype_int64, a.start64 = start.dtype == diopi_dtype_int64;
  a.new64 = fresh.dtype == diopi_dtype_int64, a.len64 = len.dtype == diopi_dtype_int64;
  a.locRowStride = loc.stride[0];
  a.kSlotStride = k.stride[0], a.kHeadStride = k.stride[1], a.vSlotStride = v.stride[0], a.vHeadStride = v.stride[1];
  a.qTok = q.stride[0], a.qHead = q.stride[1], a.oTok = out.stride[0], a.oHead = out.stride[1];
  a.slots = k.shape[0], a.rows = q.shape[0];
  a.heads = (int)q.shape[1], a.kvHeads = (int)k.shape[1], a.d = (int)q.shape[2], a.batch = (int)batch;
  a.maxNew = maxNewLen, a.maxLen = maxInputLen;
  a.scaleLog2e = kLog2eTA / sqrtf((float)a.d);
  a.group = a.heads / a.kvHeads, a.perGroup = (uint32_t)((((uint64_t)1 << 32) + a.group - 1) / a.group);
  if (pagedAttentionTiles(a, q.dtype)) return pagedAttentionMfma(ctx, stream, a, q.dtype);
  return pagedAttentionAny(stream, a, q.dtype);
}

extern "C" __attribute__((visibility("default"))) diopiError_t diopiTokenDecodeAttentionWindowInference(
    diopiContextHandle_t ctx, diopiTensorHandle_t outH, diopiConstTensorHandle_t qH, diopiConstTensorHandle_t kH,
    diopiConstTensorHandle_t vH, diopiConstTensorHandle_t locH, diopiConstTensorHandle_t startH,
    diopiConstTensorHandle_t lenH, int maxInputLen, int window, int sinks) {
  hipStream_t stream;
  AMD_TRY(getStream(ctx, &stream));
  TaViews t;
  TensorView out;
  AMD_TRY(getView(outH, &out, "out"));
  AMD_TRY(getView(qH, &t.q, "q"));
  AMD_TRY(getView(kH, &t.k, "k"));
  AMD_TRY(getView(vH, &t.v, "v"));
  AMD_TRY(getView(locH, &t.loc, "b_loc"));
  AMD_TRY(getView(startH, &t.start, "b_start_loc"));
  AMD_TRY(getView(lenH, &t.len, "b_seq_len"));
  TaArgs ta;
  AMD_TRY(fillArgs(t, true, true, maxInputLen, &ta));
  AMD_CHECK(t.q.shape[2] <= kTaGenericMaxD, "token attention: head_dim %ld exceeds %d", (long)t.q.shape[2], kTaGenericMaxD);
  AMD_CHECK(out.defined() && out.dtype == t.q.dtype && out.ndim == 3 && out.isContiguous(), "window attention: out must be a dense tensor shaped like q");
  for (int d = 0; d < 3; ++d) AMD_CHECK(out.shape[d] == t.q.shape[d], "window attention: out must be a dense tensor shaped like q");
  PaArgs a{};
  AMD_TRY(checkWindow(window, sinks, maxInputLen, &a));
  // nothing is left out: plain decode attention
  if (window == 0 || (int64_t)window + sinks >= maxInputLen) return diopiTokenDecodeAttentionInference(ctx, outH, qH, kH, vH, locH, startH, lenH, maxInputLen);
  if (t.q.numel == 0) return diopiSuccess;
  AMD_CHECK(ta.batch <= 65535, "window attention: batch %d exceeds the grid limits", ta.batch);
  if (!ta.generic) return decodeWindow(ctx, stream, ta, t.q.dtype, window, sinks, out.data);
  a.q = ta.q, a.k = ta.k, a.v = ta.v, a.out = out.data;
  a.bLoc = ta.bLoc, a.bLen = ta.bLen, a.loc64 = ta.loc64, a.len64 = ta.len64;
  a.locRowStride = ta.locRowStride;
  a.kSlotStride = ta.kSlotStride, a.kHeadStride = ta.kHeadStride, a.vSlotStride = ta.vSlotStride, a.vHeadStride = ta.vHeadStride;
  a.qTok = ta.qBatchStride, a.qHead = ta.qHeadStride, a.oTok = (int64_t)ta.heads * ta.d, a.oHead = ta.d;
  a.slots = ta.slots, a.rows = ta.batch;
  a.heads = ta.heads, a.kvHeads = ta.kvHeads, a.d = ta.d, a.batch = ta.batch, a.maxNew = 1, a.maxLen = maxInputLen;
  a.scaleLog2e = ta.scaleLog2e;
  return pagedAttentionAny(stream, a, t.q.dtype);
}
