// The int8 KV cache for gfx950: rows quantised as they are written into the pool, and read back.
//
//   k, v [tokens, kv_heads, d]          new rows (fp16, bf16 or fp32)
//   pool [slots, kv_heads, d] int8, scale [slots, kv_heads] fp32
//
// A row (one token, one head) x is kept as whole numbers q and a scale s:
//   s = max |x| / 127 rounded to fp32,  q = the whole number nearest to x / s, ties to the even one
// so q lies in [-127, 127] (it is cut to that where s has lost its last places below 2^-126). q is that of the EXACT quotient: a quotient rounded to fp32 falls on a half for one element in
// 10^5 that does not, and which neighbour it goes to would depend on how the division is done. Rows of zeros have s = 0. A row
// that holds an infinity or NaN has s = NaN and q = 0: all of it reads back as NaN, none of it as a plausible number.
// Read back: q * s rounded to fp32, and once more to a 16-bit type.
//
// Both are bound by memory: a 16-bit row of 128 moves 256 + 132 bytes.
//   * a row is spread over LPR lanes of 8 elements each (16 bytes of a 16-bit type in, 8 bytes out), so that the largest
//     magnitude is a few lane permutations; a lane asks for kKvRows rows before it works on the first;
//   * a workgroup writes the K and the V rows of its tokens, so that the tokens' destinations are looked up once.
// The last of several tokens with one destination is what the slot holds, as a loop over the tokens would leave it (a row and its
// scale must not come from two tokens). A workgroup looks through the destinations behind its own while its rows are on their
// way; above kKvScanTokens tokens, where that grows to more than the rows take, a launch of its own finds the last of each first.
#include <algorithm>

#include "common.hpp"

namespace amd {

constexpr int kKvThreads = 256;
constexpr int kKvRows = 4;               // rows that a lane group has in flight
constexpr int kKvTokensPerWg = 8;        // most tokens of a workgroup that writes
constexpr int64_t kKvScanTokens = 16384;

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
  int tokensPerWg;
  const int* last;   // the last token of each slot (null: the workgroups look for themselves)
};

__device__ __forceinline__ int64_t kvSlot(const KvInt8Args& a, int64_t t) {
  return a.loc64 ? static_cast<const int64_t*>(a.loc)[t] : static_cast<int64_t>(static_cast<const int32_t*>(a.loc)[t]);
}
// A destination counted from the end if negative; -1 outside the pool (dropped, never written).
__device__ __forceinline__ int64_t kvDestination(const KvInt8Args& a, int64_t t) {
  int64_t s = kvSlot(a, t);
  if (s < 0) s += a.slots;
  return s >= 0 && s < a.slots ? s : -1;
}

// What the magnitudes of a row and their largest (as bits: an infinity is above every number, NaN above that) make of it.
struct KvScale {
  float scale;    // what is stored
  float up;       // rows of tiny numbers are lifted by 2^64 first, so that 1 / scale is finite
  float s, inv, half;
  __device__ __forceinline__ explicit KvScale(uint32_t bits) {
    const float most = __uint_as_float(bits);
    const bool finite = bits < 0x7f800000u;
    scale = finite ? most / 127.f : __uint_as_float(0x7fc00000u);
    up = most < 0x1p-60f ? 0x1p64f : 1.f;
    s = scale * up;
    inv = finite && s > 0.f ? 1.f / s : 0.f;
    half = 0.5f * s;
  }
  // The whole number nearest to x / scale. x * inv is off by less than 2^-15, so its nearest whole number is that or a
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
  __device__ __forceinline__ float operator[](int i) const { return static_cast<float>(v[i / Vec16<T>::N][i % Vec16<T>::N]); }
};

// Which of the workgroup's tokens [t0, t0 + n) a later token supersedes, as bits (also where they have no destination).
__device__ __forceinline__ unsigned kvSuperseded(const KvInt8Args& a, int64_t t0, int n, unsigned* shared) {
  int64_t mine[kKvTokensPerWg];
  unsigned dead = 0;
#pragma unroll
  for (int i = 0; i < kKvTokensPerWg; ++i) {
    mine[i] = i < n ? kvDestination(a, t0 + i) : -1;
    if (mine[i] < 0 || (a.last != nullptr && a.last[mine[i]] != (int)(t0 + i))) dead |= 1u << i;
  }
  if (a.last != nullptr) return dead;
  if (threadIdx.x == 0) *shared = 0;
  __syncthreads();
  unsigned found = 0;
  for (int64_t j = t0 + 1 + threadIdx.x; j < a.tokens; j += kKvThreads) {
    const int64_t s = kvDestination(a, j);
#pragma unroll
    for (int i = 0; i < kKvTokensPerWg; ++i)
      if (s == mine[i] && j > t0 + i) found |= 1u << i;
  }
  if (found) atomicOr(shared, found);
  __syncthreads();
  return dead | *shared;
}

// grid: workgroups of tokensPerWg tokens. Rows of a workgroup: (pool, token, head), head fastest.
template <typename T, int LPR>
__global__ __launch_bounds__(kKvThreads) void kvInt8WriteKernel(KvInt8Args a) {
  constexpr int kGroups = kKvThreads / LPR;
  __shared__ unsigned shared;
  const int64_t t0 = (int64_t)blockIdx.x * a.tokensPerWg;
  const int n = (int)min((int64_t)a.tokensPerWg, a.tokens - t0);
  const int sub = threadIdx.x % LPR, group = threadIdx.x / LPR;
  const int rows = n * a.heads, all = 2 * rows, e = sub * 8;
  const bool live = e < a.d;
  KvPiece<T> x[kKvRows];
  auto load = [&](int r0) {
#pragma unroll
    for (int u = 0; u < kKvRows; ++u) {
      const int r = min(r0 + u * kGroups, all - 1), p = r >= rows, i = r - p * rows, t = i / a.heads, h = i - t * a.heads;
      const KvInt8Pool& o = a.pool[p];
      const T* src = static_cast<const T*>(o.x) + (t0 + t) * o.xToken + h * o.xHead + (live ? e : 0);
#pragma unroll
      for (int c = 0; c < 8 / Vec16<T>::N; ++c) x[u].v[c] = __builtin_nontemporal_load(reinterpret_cast<const typename Vec16<T>::type*>(src) + c);
    }
  };
  load(group);
  const unsigned dead = kvSuperseded(a, t0, n, &shared);
  for (int r0 = group; r0 < all; r0 += kKvRows * kGroups) {
    if (r0 != group) load(r0);
#pragma unroll
    for (int u = 0; u < kKvRows; ++u) {
      const int r = r0 + u * kGroups, p = r >= rows, i = r - p * rows, t = i / a.heads, h = i - t * a.heads;
      uint32_t most = 0;
#pragma unroll
      for (int k = 0; k < 8; ++k) most = max(most, __float_as_uint(x[u][k]) & 0x7fffffffu);
      const KvScale s(rowMost<LPR>(live ? most : 0));
      u32x2 q = {0, 0};
#pragma unroll
      for (int k = 0; k < 8; ++k) q[k / 4] |= (uint32_t)(s.nearest(x[u][k]) & 255) << (8 * (k % 4));
      if (r >= all || (dead >> t & 1)) continue;
      const KvInt8Pool& o = a.pool[p];
      const int64_t slot = kvDestination(a, t0 + t);
      if (live) *reinterpret_cast<u32x2*>(o.pool + slot * o.poolSlot + h * o.poolHead + e) = q;
      if (sub == 0) o.scale[slot * o.scaleSlot + h * o.scaleHead] = s.scale;
    }
  }
}

// Any head size and alignment: a wave per row.
template <typename T>
__global__ __launch_bounds__(kKvThreads) void kvInt8WriteAnyKernel(KvInt8Args a) {
  __shared__ unsigned shared;
  const int64_t t0 = (int64_t)blockIdx.x * a.tokensPerWg;
  const int n = (int)min((int64_t)a.tokensPerWg, a.tokens - t0);
  const unsigned dead = kvSuperseded(a, t0, n, &shared);
  const int lane = threadIdx.x & 63, rows = n * a.heads;
  for (int r = threadIdx.x / 64; r < 2 * rows; r += kKvThreads / 64) {
    const int p = r >= rows, i = r - p * rows, t = i / a.heads, h = i - t * a.heads;
    if (dead >> t & 1) continue;
    const KvInt8Pool& o = a.pool[p];
    const T* src = static_cast<const T*>(o.x) + (t0 + t) * o.xToken + h * o.xHead;
    uint32_t most = 0;
    for (int e = lane; e < a.d; e += 64) most = max(most, __float_as_uint(static_cast<float>(src[e])) & 0x7fffffffu);
    most = rowMost<32>(most);
    const KvScale s(max(most, (uint32_t)__shfl_xor((int)most, 32, 64)));
    const int64_t slot = kvDestination(a, t0 + t);
    int8_t* dst = o.pool + slot * o.poolSlot + h * o.poolHead;
    for (int e = lane; e < a.d; e += 64) dst[e] = static_cast<int8_t>(s.nearest(static_cast<float>(src[e])));
    if (lane == 0) o.scale[slot * o.scaleSlot + h * o.scaleHead] = s.scale;
  }
}

// last[slot]: the last token whose destination it is. Entries need no first value: every token writes its own to begin with,
// whichever of a slot's tokens stays there is one of them, and the largest then replaces it.
__global__ __launch_bounds__(1024) void kvInt8LastKernel(KvInt8Args a, int* last) {
  for (int64_t t = threadIdx.x; t < a.tokens; t += 1024) {
    const int64_t s = kvDestination(a, t);
    if (s >= 0) __hip_atomic_store(&last[s], (int)t, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  __threadfence();
  __syncthreads();
  for (int64_t t = threadIdx.x; t < a.tokens; t += 1024) {
    const int64_t s = kvDestination(a, t);
    if (s >= 0) __hip_atomic_fetch_max(&last[s], (int)t, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
}

// grid: workgroups of tokensPerWg rows of `loc` (K and V)
template <typename T, int LPR>
__global__ __launch_bounds__(kKvThreads) void kvInt8ReadKernel(KvInt8Args a) {
  constexpr int kGroups = kKvThreads / LPR;
  const int64_t t0 = (int64_t)blockIdx.x * a.tokensPerWg;
  const int n = (int)min((int64_t)a.tokensPerWg, a.tokens - t0);
  const int sub = threadIdx.x % LPR, group = threadIdx.x / LPR;
  const int rows = n * a.heads, all = 2 * rows, e = sub * 8;
  if (e >= a.d) return;
  for (int r0 = group; r0 < all; r0 += kKvRows * kGroups) {
    u32x2 q[kKvRows];
    float s[kKvRows];
#pragma unroll
    for (int u = 0; u < kKvRows; ++u) {
      const int r = min(r0 + u * kGroups, all - 1), p = r >= rows, i = r - p * rows, t = i / a.heads, h = i - t * a.heads;
      const KvInt8Pool& o = a.pool[p];
      const int64_t slot = kvSlot(a, t0 + t);
      const bool in = slot >= 0 && slot < a.slots;  // outside the pool: zeros, nothing is read
      q[u] = u32x2{0, 0}, s[u] = 0.f;
      if (in) {
        q[u] = __builtin_nontemporal_load(reinterpret_cast<const u32x2*>(o.pool + slot * o.poolSlot + h * o.poolHead + e));
        s[u] = o.scale[slot * o.scaleSlot + h * o.scaleHead];
      }
    }
#pragma unroll
    for (int u = 0; u < kKvRows; ++u) {
      const int r = r0 + u * kGroups, p = r >= rows, i = r - p * rows, t = i / a.heads, h = i - t * a.heads;
      if (r >= all) continue;
      KvPiece<T> x;
#pragma unroll
      for (int k = 0; k < 8; ++k)
        x.v[k / Vec16<T>::N][k % Vec16<T>::N] = static_cast<T>(static_cast<float>((int)(q[u][k / 4] << (24 - 8 * (k % 4))) >> 24) * s[u]);
      const KvInt8Pool& o = a.pool[p];
      T* dst = static_cast<T*>(o.x) + (t0 + t) * o.xToken + h * o.xHead + e;
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
  for (int r = threadIdx.x / 64; r < 2 * rows; r += kKvThreads / 64) {
    const int p = r >= rows, i = r - p * rows, t = i / a.heads, h = i - t * a.heads;
    const KvInt8Pool& o = a.pool[p];
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
  a->heads = (int)x[0].shape[1], a->d = (int)x[0].shape[2];
  a->last = nullptr;
  return diopiSuccess;
}

// Whether all rows lie in whole 8-element pieces that can be loaded and stored at once.
static bool kvInt8Vector(const KvInt8Args& a, int64_t itemsize) {
  if (a.d % 8 != 0 || a.d > 256) return false;
  int64_t bits16 = 0, bits8 = 0;
  for (const KvInt8Pool& o : a.pool) {
    bits16 |= (int64_t)reinterpret_cast<uintptr_t>(o.x) | o.xToken * itemsize | o.xHead * itemsize;
    bits8 |= (int64_t)reinterpret_cast<uintptr_t>(o.pool) | o.poolSlot | o.poolHead;
  }
  return (bits16 & 15) == 0 && (bits8 & 7) == 0;
}

#define KV_INT8_LAUNCH_TYPE(T, NAME, VEC)                                                                            \
  do {                                                                                                               \
    if (!(VEC)) hipLaunchKernelGGL((NAME##AnyKernel<T>), grid, dim3(kKvThreads), 0, stream, a);                       \
    else if (a.d <= 64) hipLaunchKernelGGL((NAME##Kernel<T, 8>), grid, dim3(kKvThreads), 0, stream, a);               \
    else if (a.d <= 128) hipLaunchKernelGGL((NAME##Kernel<T, 16>), grid, dim3(kKvThreads), 0, stream, a);             \
    else hipLaunchKernelGGL((NAME##Kernel<T, 32>), grid, dim3(kKvThreads), 0, stream, a);                             \
  } while (0)
#define KV_INT8_LAUNCH(DTYPE, NAME, VEC)                                          \
  do {                                                                            \
    if (DTYPE == diopi_dtype_bfloat16) KV_INT8_LAUNCH_TYPE(bf16_t, NAME, VEC);    \
    else if (DTYPE == diopi_dtype_float16) KV_INT8_LAUNCH_TYPE(half_t, NAME, VEC); \
    else KV_INT8_LAUNCH_TYPE(float, NAME, VEC);                                   \
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
  AMD_TRY(makeContiguous(ctx, stream, loc, &dense));
  a.loc = dense.data;
  if (a.tokens > kKvScanTokens) {
    AMD_CHECK(a.slots < ((int64_t)1 << 31), "%s: %ld slots exceed 2^31 - 1", what, (long)a.slots);
    void* last = nullptr;
    AMD_TRY(requireWorkspace(ctx, a.slots * (int64_t)sizeof(int), &last));
    hipLaunchKernelGGL(kvInt8LastKernel, dim3(1), dim3(1024), 0, stream, a, static_cast<int*>(last));
    AMD_LAUNCH_CHECK();
    a.last = static_cast<const int*>(last);
  }
  a.tokensPerWg = (int)std::min<int64_t>(kKvTokensPerWg, std::max<int64_t>(1, a.tokens / 1024));
  const dim3 grid((unsigned)ceilDiv(a.tokens, a.tokensPerWg));
  KV_INT8_LAUNCH(x[0].dtype, kvInt8Write, kvInt8Vector(a, x[0].itemsize));
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
  AMD_TRY(makeContiguous(ctx, stream, loc, &dense));
  a.loc = dense.data;
  a.tokensPerWg = (int)std::min<int64_t>(kKvTokensPerWg, std::max<int64_t>(1, a.tokens / 1024));
  const dim3 grid((unsigned)ceilDiv(a.tokens, a.tokensPerWg));
  KV_INT8_LAUNCH(x[0].dtype, kvInt8Read, kvInt8Vector(a, x[0].itemsize));
  AMD_LAUNCH_CHECK();
  return diopiSuccess;
}
