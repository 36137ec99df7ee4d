// Slot-mapping scatter of fresh K/V rows into an e4m3 paged cache with one
// scale for each block of G tokens and KV head.
//
//     scale   = 2^e, the smallest power of two with amax <= 448 * scale over
//               the block's finite values, e >= -100
//     payload = e4m3_rne(x / scale); a value that is not finite becomes NaN
//
// The scale is a power of two because blocks grow: a decode step adds one
// token to a block that holds others, and when the token needs a larger scale
// the other rows are written again. By a power of two that is exact but for
// values that fall among the subnormals (steps of 2^-9 of the scale), however
// often it happens, where a scale of amax/448 would add a rounding of up to
// 2^-4 each time. It costs no precision: e4m3 is a floating-point format, and
// a block whose largest payload is 224 instead of 448 keeps the same relative
// steps.
//
// A call that writes a block's first token opens the block: its old scale and
// rows no longer count (the rows keep their bytes). Otherwise the new scale is
// the larger of the old one and what the call's rows need, and the rows that
// the call does not write are multiplied by old / new. An old scale that is
// not a positive finite number counts as zero.
//
// The slots of a call come in any order, and a slot that occurs twice takes
// the later row, so the result does not depend on timing: one CTA owns a
// block. The first token of a run of tokens in one block reads all slots of
// the call, from L2; if an earlier token has the same block its CTA leaves,
// else it has every row of the block and the last writer of each. That is a
// quadratic number of slot reads, 4 bytes each against 6 KB of K and V a
// token; runs are as long as blocks in a prompt, so at 16384 tokens it is
// 64 KB for each 64 KB of rows (one in sixteen tokens begins a run), out of
// L2. A sort or a workspace of claims would cost another launch, which is
// more than the whole store of a decode step.
//
// The rest is memory bound: 2 bytes read and 1 written per value. LANES
// threads hold a row, 8 values (one 16-byte load, one 8-byte store) each. A
// CTA takes `pairs` (K or V, head) pairs of the block and deals the block's
// rows over the thread groups of each pair.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "codec.cuh"
#include "runtime.h"

namespace kvoff {
namespace {

constexpr int kThreads = 256;
constexpr int kKept = 4;        // rows of a thread group held in registers between the passes
constexpr int kWindow = 16;     // tokens a CTA looks at for the start of a run
constexpr int64_t kSmallCall = 1024;  // up to here a CTA looks at one token
constexpr int64_t kMostTokens = 65536;
constexpr int kMostBlock = 4096;
constexpr int kMinExponent = -100;

struct StoreArgs {
  const uint8_t* rows[2];  // key, value
  int64_t stride[2];       // bytes per token
  uint8_t* cache[2];
  float* scale[2];
  const int32_t* slots;
  int32_t* bad_slots;
  int64_t num_slots;
  int32_t num_tokens, heads, dim, shift, pairs, window;
  bool wide_slots;  // slots can be read 16 bytes at a time
};

template <typename T>
__device__ __forceinline__ void unpack(const uint4& v, float (&x)[8]);
template <>
__device__ __forceinline__ void unpack<__nv_bfloat16>(const uint4& v, float (&x)[8]) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = __uint_as_float(w[i] << 16);
    x[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
  }
}
template <>
__device__ __forceinline__ void unpack<__half>(const uint4& v, float (&x)[8]) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
    x[2 * i] = f.x;
    x[2 * i + 1] = f.y;
  }
}

// Bits of the largest finite magnitude among the values, and `most`.
__device__ __forceinline__ uint32_t finite_amax(const float (&x)[8], uint32_t most) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t m = __float_as_uint(x[i]) & 0x7FFFFFFFu;
    if (m < 0x7F800000u) most = max(most, m);
  }
  return most;
}

// The smallest power of two s with amax <= 448 s = 1.75 * 2^8 s, at least 2^kMinExponent.
__device__ __forceinline__ float scale_for(uint32_t amax_bits) {
  int e = (int)(amax_bits >> 23) - 127 - 8 + ((amax_bits & 0x7FFFFFu) > 0x600000u);
  e = max(e, kMinExponent);
  return __uint_as_float((uint32_t)(e + 127) << 23);
}

// x / scale as e4m3 bytes. The reciprocal of a power of two is exact; another
// scale (one that the caller put there) is divided by.
__device__ __forceinline__ uint2 encode(const float (&x)[8], float scale) {
  float y[8];
  if ((__float_as_uint(scale) & 0x7FFFFFu) == 0) {
    const float r = __fdiv_rn(1.0f, scale);
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = x[i] * r;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = __fdiv_rn(x[i], scale);
  }
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if ((__float_as_uint(x[i]) & 0x7FFFFFFFu) >= 0x7F800000u) y[i] = __uint_as_float(0x7FC00000u);
  uint2 out;
  out.x = f32x2_to_e4m3x2(y[0], y[1]) | f32x2_to_e4m3x2(y[2], y[3]) << 16;
  out.y = f32x2_to_e4m3x2(y[4], y[5]) | f32x2_to_e4m3x2(y[6], y[7]) << 16;
  return out;
}

__device__ __forceinline__ uint2 rescale(const uint2& payload, float factor) {
  const float2 a = e4m3x2_to_f32x2(payload.x & 0xFFFFu), b = e4m3x2_to_f32x2(payload.x >> 16);
  const float2 c = e4m3x2_to_f32x2(payload.y & 0xFFFFu), d = e4m3x2_to_f32x2(payload.y >> 16);
  uint2 out;
  out.x = f32x2_to_e4m3x2(a.x * factor, a.y * factor) |
          f32x2_to_e4m3x2(b.x * factor, b.y * factor) << 16;
  out.y = f32x2_to_e4m3x2(c.x * factor, c.y * factor) |
          f32x2_to_e4m3x2(d.x * factor, d.y * factor) << 16;
  return out;
}

template <typename T, int LANES>
__global__ void __launch_bounds__(kThreads) store_kvcache_fp8_kernel(const StoreArgs a) {
  constexpr int kGroups = kThreads / LANES;
  extern __shared__ int32_t shared[];
  __shared__ int32_t window[kWindow + 1];
  __shared__ uint32_t amax[kGroups];
  __shared__ int32_t count, earlier;
  const int block = 1 << a.shift;
  int32_t* winner = shared;          // last token that writes each row of the block, or -1
  int32_t* written = shared + block;  // the rows that have one
  const int tid = threadIdx.x, lane = tid % LANES;
  const int mine = (tid / LANES) % a.pairs;  // this thread's pair among the CTA's
  const int sub = (tid / LANES) / a.pairs, subs = kGroups / a.pairs;
  const int pair = blockIdx.y * a.pairs + mine;
  const bool active = pair < 2 * a.heads && lane * 8 < a.dim;
  const int kv = pair >= a.heads ? 1 : 0, head = pair - kv * a.heads;
  const int64_t row_bytes = (int64_t)a.heads * a.dim;
  const int first = blockIdx.x * a.window;

  // slot_mapping[first - 1 .. first + window): is a token the start of a run?
  if (tid <= a.window) {
    const int i = first - 1 + tid;
    int32_t slot = -1;
    if (i >= 0 && i < a.num_tokens) slot = a.slots[i];
    if (slot >= a.num_slots) {
      if (tid > 0 && blockIdx.y == 0 && a.bad_slots != nullptr) atomicAdd(a.bad_slots, 1);
      slot = -1;
    }
    window[tid] = slot < 0 ? -1 : slot >> a.shift;
  }
  __syncthreads();

  for (int w = 1; w <= a.window; ++w) {
    const int32_t id = window[w];
    if (id < 0 || id == window[w - 1]) continue;  // the same decision in all threads
    const int leader = first + w - 1;
    for (int i = tid; i < block; i += kThreads) winner[i] = -1;
    if (tid < a.pairs) amax[tid] = 0;
    if (tid == 0) count = earlier = 0;
    __syncthreads();
    const int64_t base = (int64_t)id << a.shift;
    auto look = [&](int i, int32_t slot) {
      if (slot >= 0 && slot >> a.shift == id) {
        if (i < leader)
          earlier = 1;
        else
          atomicMax(&winner[slot - (int32_t)base], i);
      }
    };
    if (a.wide_slots) {
      const int quads = a.num_tokens / 4;
      for (int i = tid; i < quads; i += kThreads) {
        const int4 s = __ldg(reinterpret_cast<const int4*>(a.slots) + i);
        look(4 * i, s.x);
        look(4 * i + 1, s.y);
        look(4 * i + 2, s.z);
        look(4 * i + 3, s.w);
      }
      for (int i = 4 * quads + tid; i < a.num_tokens; i += kThreads) look(i, __ldg(a.slots + i));
    } else {
      for (int i = tid; i < a.num_tokens; i += kThreads) look(i, __ldg(a.slots + i));
    }
    __syncthreads();
    if (earlier != 0) {  // another CTA owns the block
      __syncthreads();
      continue;
    }
    for (int i = tid; i < block; i += kThreads)
      if (winner[i] >= 0) written[atomicAdd(&count, 1)] = i;
    const bool opened = winner[0] >= 0;
    float* scale = (kv != 0 ? a.scale[1] : a.scale[0]) + (int64_t)id * a.heads + head;
    float old = 0.0f;
    if (active && !opened) {
      old = *scale;
      if (!(old > 0.0f && __float_as_uint(old) < 0x7F800000u)) old = 0.0f;
    }
    __syncthreads();

    const int rows = count;
    const int64_t stride = kv != 0 ? a.stride[1] : a.stride[0];
    const uint8_t* source =
        (kv != 0 ? a.rows[1] : a.rows[0]) + ((int64_t)head * a.dim + lane * 8) * sizeof(T);
    uint8_t* target = (kv != 0 ? a.cache[1] : a.cache[0]) + base * row_bytes + (int64_t)head * a.dim + lane * 8;
    uint32_t most = 0;
    uint4 kept[kKept];
    if (active) {
#pragma unroll
      for (int i = 0; i < kKept; ++i) {
        const int r = sub + i * subs;
        if (r < rows)
          kept[i] = *reinterpret_cast<const uint4*>(source + winner[written[r]] * stride);
      }
#pragma unroll
      for (int i = 0; i < kKept; ++i)
        if (sub + i * subs < rows) {
          float x[8];
          unpack<T>(kept[i], x);
          most = finite_amax(x, most);
        }
#pragma unroll 4
      for (int r = sub + kKept * subs; r < rows; r += subs) {
        float x[8];
        unpack<T>(*reinterpret_cast<const uint4*>(source + winner[written[r]] * stride), x);
        most = finite_amax(x, most);
      }
    }
#pragma unroll
    for (int d = LANES / 2; d > 0; d /= 2) most = max(most, __shfl_xor_sync(0xFFFFFFFFu, most, d));
    if (lane == 0 && most != 0) atomicMax(&amax[mine], most);
    __syncthreads();
    if (active) {
      const float now = fmaxf(scale_for(amax[mine]), old);
#pragma unroll
      for (int i = 0; i < kKept; ++i) {
        const int r = sub + i * subs;
        if (r < rows) {
          float x[8];
          unpack<T>(kept[i], x);
          *reinterpret_cast<uint2*>(target + written[r] * row_bytes) = encode(x, now);
        }
      }
#pragma unroll 4
      for (int r = sub + kKept * subs; r < rows; r += subs) {
        float x[8];
        unpack<T>(*reinterpret_cast<const uint4*>(source + winner[written[r]] * stride), x);
        *reinterpret_cast<uint2*>(target + written[r] * row_bytes) = encode(x, now);
      }
      if (!opened && now != old) {
        const float factor = __fdiv_rn(old, now);
        for (int r = sub; r < block; r += subs)
          if (winner[r] < 0) {
            uint2* p = reinterpret_cast<uint2*>(target + r * row_bytes);
            *p = rescale(*p, factor);
          }
      }
      if (sub == 0 && lane == 0) *scale = now;
    }
    __syncthreads();
  }
}

template <typename T, int LANES>
int launch(StoreArgs a, cudaStream_t stream) {
  constexpr int kGroups = kThreads / LANES;
  const int block = 1 << a.shift;
  a.window = a.num_tokens <= kSmallCall ? 1 : kWindow;
  // As many pairs a CTA as it has thread groups, fewer while that leaves SMs
  // without a block (a prompt of one sequence in long blocks).
  const int64_t blocks = a.num_tokens <= kSmallCall && a.num_tokens < block
                             ? a.num_tokens
                             : (a.num_tokens + block - 1) / block;
  int pairs = 1;
  while (pairs < kGroups && pairs < 2 * a.heads) pairs *= 2;
  while (pairs > 1 && blocks * ((2 * a.heads + pairs - 1) / pairs) < 4 * sm_count()) pairs /= 2;
  a.pairs = pairs;
  const dim3 grid((a.num_tokens + a.window - 1) / a.window, (2 * a.heads + pairs - 1) / pairs);
  store_kvcache_fp8_kernel<T, LANES>
      <<<grid, kThreads, 2 * block * sizeof(int32_t), stream>>>(a);
  return cuda_status(cudaGetLastError(), "store_kvcache_fp8 launch");
}

template <typename T>
int launch_lanes(const StoreArgs& a, cudaStream_t stream) {
  const int vectors = a.dim / 8;
  if (vectors <= 4) return launch<T, 4>(a, stream);
  if (vectors <= 8) return launch<T, 8>(a, stream);
  if (vectors <= 16) return launch<T, 16>(a, stream);
  return launch<T, 32>(a, stream);
}

}  // namespace
}  // namespace kvoff

using namespace kvoff;

extern "C" int kvoff_store_kvcache_fp8(const void* key, int64_t key_stride_bytes,
                                       const void* value, int64_t value_stride_bytes,
                                       void* k_cache, void* v_cache, float* k_scale,
                                       float* v_scale, int64_t num_heads, int64_t head_dim,
                                       int32_t dtype, int64_t scale_block,
                                       const int32_t* slot_mapping, int64_t num_tokens,
                                       int64_t num_slots, int32_t* bad_slots, void* stream) {
  if (injected("store_kvcache_fp8")) return KVOFF_EINJECTED;
  if (num_tokens < 0 || num_heads <= 0 || num_heads > 32767 || num_slots < 0 ||
      key_stride_bytes < 0 || value_stride_bytes < 0)
    return fail(KVOFF_EINVAL, "kvoff_store_kvcache_fp8: bad sizes");
  if (head_dim <= 0 || head_dim % 8 != 0 || head_dim > 256)
    return fail(KVOFF_EINVAL, "kvoff_store_kvcache_fp8: head_dim %lld is not a multiple of 8 up to 256",
                (long long)head_dim);
  if (dtype != KVOFF_BF16 && dtype != KVOFF_FP16)
    return fail(KVOFF_EINVAL, "kvoff_store_kvcache_fp8: rows are bf16 or fp16");
  if (scale_block <= 0 || (scale_block & (scale_block - 1)) != 0 || scale_block > kMostBlock ||
      num_slots % scale_block != 0)
    return fail(KVOFF_EINVAL,
                "kvoff_store_kvcache_fp8: a scale block is a power of two up to %d tokens that "
                "divides the cache",
                kMostBlock);
  if (num_slots > 0x7FFFFFFFll)
    return fail(KVOFF_EINVAL, "kvoff_store_kvcache_fp8: slots are int32");
  if (num_tokens == 0) return ok();
  if (num_tokens > kMostTokens)
    return fail(KVOFF_EINVAL, "kvoff_store_kvcache_fp8: %lld tokens exceed one call's %lld",
                (long long)num_tokens, (long long)kMostTokens);
  if (key == nullptr || value == nullptr || k_cache == nullptr || v_cache == nullptr ||
      k_scale == nullptr || v_scale == nullptr || slot_mapping == nullptr)
    return fail(KVOFF_EINVAL, "kvoff_store_kvcache_fp8: null pointer");
  const uintptr_t wide = reinterpret_cast<uintptr_t>(key) | reinterpret_cast<uintptr_t>(value) |
                         (uintptr_t)key_stride_bytes | (uintptr_t)value_stride_bytes;
  const uintptr_t narrow = reinterpret_cast<uintptr_t>(k_cache) | reinterpret_cast<uintptr_t>(v_cache);
  if ((wide & 15u) != 0 || (narrow & 7u) != 0)
    return fail(KVOFF_EINVAL,
                "kvoff_store_kvcache_fp8: rows must be 16-byte aligned and caches 8-byte aligned");
  StoreArgs a{};
  a.rows[0] = static_cast<const uint8_t*>(key);
  a.rows[1] = static_cast<const uint8_t*>(value);
  a.stride[0] = key_stride_bytes;
  a.stride[1] = value_stride_bytes;
  a.cache[0] = static_cast<uint8_t*>(k_cache);
  a.cache[1] = static_cast<uint8_t*>(v_cache);
  a.scale[0] = k_scale;
  a.scale[1] = v_scale;
  a.slots = slot_mapping;
  a.bad_slots = bad_slots;
  a.num_slots = num_slots;
  a.num_tokens = (int32_t)num_tokens;
  a.heads = (int32_t)num_heads;
  a.dim = (int32_t)head_dim;
  a.wide_slots = (reinterpret_cast<uintptr_t>(slot_mapping) & 15u) == 0;
  while ((1ll << a.shift) < scale_block) ++a.shift;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int rc = dtype == KVOFF_BF16 ? launch_lanes<__nv_bfloat16>(a, s) : launch_lanes<__half>(a, s);
  if (rc != KVOFF_OK) return rc;
  return ok();
}
