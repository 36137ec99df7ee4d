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
// the call; if an earlier token has the same block its CTA leaves, else it has
// every row of the block and the last writer of each. That is a quadratic
// number of slot reads, 4 bytes each against 6 KB of K and V a token, out of
// L1 for all but the first CTAs of an SM: 4 of 41 us for 16384 tokens in blocks
// of 16. A sort or a workspace of claims would cost another launch, which is
// more than the whole store of a decode step.
//
// The rest is memory bound: 2 bytes read and 1 written per value. LANES
// threads hold a row, 8 values (one 16-byte load, one 8-byte store) each. A
// CTA takes `pairs` (K or V, head) pairs of the block and deals the block's
// rows over the thread groups of each pair. In a large call, which holds
// prompts, a run's rows are on the way while the slots are looked at.
//
// Measured: 4096 tokens, 8 heads of 128, blocks of 64 in 14 us (3.8 us at a
// copy's rate), 16384 ragged tokens in blocks of 16 in 41 us (15.4), 4 tokens
// in 3.3 us. What bounds it is the chain of a CTA: slots of its window, rows,
// three barriers, the scale, the writes. 256 threads a CTA in the large call
// take 46 us, 128 registers instead of 64 and half the CTAs 42 us.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "codec.cuh"
#include "runtime.h"

namespace kvoff {
namespace {

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
  int32_t num_tokens, heads, dim, shift, pairs, pair_shift, window;
  bool wide_slots;  // slots can be read 16 bytes at a time
};

// Both rows' types order their magnitudes by their bits; from kInf on they are
// infinities and NaN.
template <typename T>
constexpr uint32_t kInf = std::is_same<T, __half>::value ? 0x7C00u : 0x7F80u;

template <typename T>
__device__ __forceinline__ float2 unpack(uint32_t w) {
  if constexpr (std::is_same<T, __half>::value)
    return __half22float2(*reinterpret_cast<const __half2*>(&w));
  else
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
}

// Magnitude bits (16) of the largest of the eight values.
__device__ __forceinline__ uint32_t largest(const uint4& v) {
  constexpr uint32_t m = 0x7FFF7FFFu;
  const uint32_t x = __vmaxu2(__vmaxu2(v.x & m, v.y & m), __vmaxu2(v.z & m, v.w & m));
  return max(x & 0xFFFFu, x >> 16);
}

// The same among the finite values.
template <typename T>
__device__ __noinline__ uint32_t largest_finite(uint4 v) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
  uint32_t most = 0;
  for (int i = 0; i < 8; ++i) {
    const uint32_t m = w[i / 2] >> i % 2 * 16 & 0x7FFFu;
    if (m < kInf<T>) most = max(most, m);
  }
  return most;
}

// The smallest power of two s with amax <= 448 s = 1.75 * 2^8 s, at least 2^kMinExponent.
template <typename T>
__device__ __forceinline__ float scale_for(uint32_t amax16) {
  const uint32_t bits = __float_as_uint(unpack<T>(amax16).x);
  int e = (int)(bits >> 23) - 127 - 8 + ((bits & 0x7FFFFFu) > 0x600000u);
  e = max(e, kMinExponent);
  return __uint_as_float((uint32_t)(e + 127) << 23);
}

// x / scale as e4m3 bytes, NaN where x is not finite. The reciprocal of a power
// of two is exact; another scale (one that the caller put there) is divided by.
template <typename T>
__device__ __noinline__ uint2 encode_any(uint4 v, float scale) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
  uint32_t out[4];
  for (int i = 0; i < 4; ++i) {
    const float2 x = unpack<T>(w[i]);
    const float nan = __uint_as_float(0x7FC00000u);
    const float lo = (w[i] & 0x7FFFu) < kInf<T> ? __fdiv_rn(x.x, scale) : nan;
    const float hi = (w[i] >> 16 & 0x7FFFu) < kInf<T> ? __fdiv_rn(x.y, scale) : nan;
    out[i] = f32x2_to_e4m3x2(lo, hi);
  }
  return make_uint2(out[0] | out[1] << 16, out[2] | out[3] << 16);
}

template <typename T>
__device__ __forceinline__ uint2 encode_finite(const uint4& v, float reciprocal) {
  const float2 a = unpack<T>(v.x), b = unpack<T>(v.y), c = unpack<T>(v.z), d = unpack<T>(v.w);
  const float r = reciprocal;
  uint2 out;
  out.x = f32x2_to_e4m3x2(a.x * r, a.y * r) | f32x2_to_e4m3x2(b.x * r, b.y * r) << 16;
  out.y = f32x2_to_e4m3x2(c.x * r, c.y * r) | f32x2_to_e4m3x2(d.x * r, d.y * r) << 16;
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

__device__ __forceinline__ uint4 load_row(const uint8_t* p) {
  uint4 v;  // read once: kept out of L1, which holds the slots
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p));
  return v;
}

template <typename T, int LANES, int THREADS, int KEPT>
__global__ void __launch_bounds__(THREADS, 1024 / THREADS)
    store_kvcache_fp8_kernel(const __grid_constant__ StoreArgs a) {
  constexpr int kGroups = THREADS / LANES;
  extern __shared__ int32_t winner[];  // last token that writes each row of the block, or -1
  __shared__ int32_t window[kWindow];
  __shared__ uint32_t starts;
  __shared__ uint32_t amax[kGroups];
  __shared__ int32_t earlier, last;
  const int tid = threadIdx.x;
  const int first = blockIdx.x * a.window;

  // Which of the CTA's tokens begin a run: those whose nearest token before
  // them, skipped ones left out, is in another block (or is not looked at).
  if (tid < 32) {
    const int i = first - (32 - kWindow) + tid;  // lanes 16 .. 16 + window: the CTA's tokens
    const bool own = tid >= 32 - kWindow && tid < 32 - kWindow + a.window;
    int32_t slot = -1;
    if (i >= 0 && i < a.num_tokens) slot = __ldg(a.slots + i);
    if (slot >= a.num_slots) {
      if (own && blockIdx.y == 0 && a.bad_slots != nullptr) atomicAdd(a.bad_slots, 1);
      slot = -1;
    }
    const int32_t id = slot < 0 ? -1 : slot >> a.shift;
    const uint32_t before = __ballot_sync(0xFFFFFFFFu, id >= 0) & ((1u << tid) - 1);
    const int32_t previous = __shfl_sync(0xFFFFFFFFu, id, before == 0 ? 0 : 31 - __clz(before));
    const bool start = own && id >= 0 && (before == 0 || previous != id);
    const uint32_t mask = __ballot_sync(0xFFFFFFFFu, start) >> (32 - kWindow);
    if (own) window[tid - (32 - kWindow)] = slot;
    if (tid == 0) starts = mask;
  }
  __syncthreads();
  uint32_t todo = starts;
  if (todo == 0) return;

  const uint32_t block = 1u << a.shift;
  const int lane = tid % LANES;
  const int mine = (tid / LANES) & (a.pairs - 1);  // this thread's pair among the CTA's
  const int subs = kGroups >> a.pair_shift, sub = (tid / LANES) >> a.pair_shift;
  const int pair = blockIdx.y * a.pairs + mine;
  const bool active = pair < 2 * a.heads && lane * 8 < a.dim;
  const bool is_v = pair >= a.heads;
  const int head = is_v ? pair - a.heads : pair;
  const int64_t row_bytes = (int64_t)a.heads * a.dim;
  const int64_t stride = is_v ? a.stride[1] : a.stride[0];
  const uint8_t* source =
      (is_v ? a.rows[1] : a.rows[0]) + ((int64_t)head * a.dim + lane * 8) * sizeof(T);
  for (; todo != 0; todo &= todo - 1) {
    const int w = __ffs(todo) - 1, leader = first + w;
    const int32_t id = window[w] >> a.shift, base = id << a.shift;
    const int32_t begin = window[w] - base;  // the leader's row
    for (int i = tid; i < (int)block; i += THREADS) winner[i] = -1;
    if (tid < a.pairs) amax[tid] = 0;
    if (tid == 0) earlier = last = 0;
    // Rows that are nearly always the block's are on the way while the slots are
    // looked at: those of the tokens after the leader in a large call, which
    // holds prompts; the leader's own in a small one.
    const uint8_t* run = source + (leader + sub) * stride;
    const int likely = a.window > 1 ? min((int)block - begin, a.num_tokens - leader) : 1;
    uint4 kept[KEPT];
#pragma unroll
    for (int i = 0; i < KEPT; ++i)
      if (active && sub + i * subs < likely) kept[i] = load_row(run + i * subs * stride);
    float* scale = (is_v ? a.scale[1] : a.scale[0]) + (int64_t)id * a.heads + head;
    float before = 0.0f;
    if (active) before = *scale;
    __syncthreads();
    // A slot's row in the block, or a number not below `block`.
    auto row_of = [&](int32_t slot) { return (uint32_t)slot - (uint32_t)base; };
    auto look = [&](int i, int32_t slot) {
      if (row_of(slot) < block) {
        if (i < leader)
          earlier = 1;
        else
          atomicMax(&winner[row_of(slot)], i);
      }
    };
    if (a.wide_slots) {
      const int quads = a.num_tokens / 4;
#pragma unroll 4
      for (int i = tid; i < quads; i += THREADS) {
        const int4 s = __ldg(reinterpret_cast<const int4*>(a.slots) + i);
        if (min(min(row_of(s.x), row_of(s.y)), min(row_of(s.z), row_of(s.w))) < block) {
          look(4 * i, s.x);
          look(4 * i + 1, s.y);
          look(4 * i + 2, s.z);
          look(4 * i + 3, s.w);
        }
      }
      for (int i = 4 * quads + tid; i < a.num_tokens; i += THREADS) look(i, __ldg(a.slots + i));
    } else {
      for (int i = tid; i < a.num_tokens; i += THREADS) look(i, __ldg(a.slots + i));
    }
    __syncthreads();
    if (earlier != 0) {  // another CTA owns the block
      __syncthreads();
      continue;
    }
    // The usual case: tokens that follow one another write rows that follow one
    // another (some may be skipped), up to `extent` of them from `begin` on, and no
    // other token writes here.
    bool in_order = true;
    int most_row = 0;
    for (int i = tid; i < (int)block; i += THREADS)
      if (winner[i] >= 0) {
        in_order = in_order && winner[i] - leader == i - begin;
        most_row = i + 1;
      }
    most_row = __reduce_max_sync(0xFFFFFFFFu, most_row);
    if (tid % 32 == 0 && most_row > 0) atomicMax(&last, most_row);
    const bool regular = __syncthreads_and(in_order);
    const int extent = last - begin;
    const bool opened = winner[0] >= 0;
    const float old =
        !opened && before > 0.0f && __float_as_uint(before) < 0x7F800000u ? before : 0.0f;

    uint8_t* target = (is_v ? a.cache[1] : a.cache[0]) + base * row_bytes +
                      (int64_t)head * a.dim + lane * 8;
    // Calls f(row, its number in the block) for this thread's rows that are not
    // in `kept`.
    auto others = [&](auto f) {
      if (regular) {
#pragma unroll 4
        for (int r = sub + KEPT * subs; r < extent; r += subs)
          if (winner[begin + r] >= 0) f(load_row(source + (leader + r) * stride), begin + r);
      } else {
        for (int r = sub; r < (int)block; r += subs)
          if (winner[r] >= 0) f(load_row(source + winner[r] * stride), r);
      }
    };
    uint32_t most = 0;
    bool finite = true;
    auto size_of = [&](const uint4& row) {
      const uint32_t size = largest(row);
      if (size < kInf<T>) return size;
      finite = false;
      return largest_finite<T>(row);
    };
    uint32_t held = 0;  // bit i: kept[i] is written
    if (active) {
#pragma unroll
      for (int i = 0; i < KEPT; ++i) {
        const int r = sub + i * subs;
        if (regular && r < extent && winner[begin + r] >= 0) {
          held |= 1u << i;
          if (r >= likely) kept[i] = load_row(run + i * subs * stride);
        }
      }
#pragma unroll
      for (int i = 0; i < KEPT; ++i)
        if (held >> i & 1) most = max(most, size_of(kept[i]));
      others([&](const uint4& row, int) { most = max(most, size_of(row)); });
    }
#pragma unroll
    for (int d = LANES / 2; d > 0; d /= 2) most = max(most, __shfl_xor_sync(0xFFFFFFFFu, most, d));
    if (lane == 0 && most != 0) atomicMax(&amax[mine], most);
    __syncthreads();
    if (active) {
      const float now = fmaxf(scale_for<T>(amax[mine]), old);
      const float reciprocal = __fdiv_rn(1.0f, now);
      const bool plain = finite && (__float_as_uint(now) & 0x7FFFFFu) == 0;
      auto put = [&](const uint4& row, uint8_t* to) {
        *reinterpret_cast<uint2*>(to) = plain ? encode_finite<T>(row, reciprocal) : encode_any<T>(row, now);
      };
      uint8_t* to = target + (begin + sub) * row_bytes;
#pragma unroll
      for (int i = 0; i < KEPT; ++i) {
        if (held >> i & 1) put(kept[i], to);
        to += subs * row_bytes;
      }
      others([&](const uint4& row, int at) { put(row, target + at * row_bytes); });
      if (!opened && now != old) {
        const float factor = __fdiv_rn(old, now);
        for (int r = sub; r < (int)block; r += subs)
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

template <typename T, int LANES, int THREADS, int KEPT>
int launch(StoreArgs a, cudaStream_t stream) {
  constexpr int kGroups = THREADS / LANES;
  const int block = 1 << a.shift;
  a.window = a.num_tokens <= kSmallCall ? 1 : kWindow;
  // As many pairs a CTA as it has thread groups; fewer while that leaves SMs
  // without a block (a prompt of one sequence in long blocks), or while a group
  // has more rows than it holds in registers.
  const int64_t blocks = a.num_tokens <= kSmallCall && a.num_tokens < block
                             ? a.num_tokens
                             : (a.num_tokens + block - 1) / block;
  int pairs = 1;
  while (pairs < kGroups && pairs < 2 * a.heads) pairs *= 2;
  while (pairs > 1 && (blocks * ((2 * a.heads + pairs - 1) / pairs) < sm_count() ||
                       kGroups / pairs * KEPT < (a.window > 1 ? block : 1)))
    pairs /= 2;
  a.pairs = pairs;
  while ((1 << a.pair_shift) < pairs) ++a.pair_shift;
  const dim3 grid((a.num_tokens + a.window - 1) / a.window, (2 * a.heads + pairs - 1) / pairs);
  store_kvcache_fp8_kernel<T, LANES, THREADS, KEPT>
      <<<grid, THREADS, block * sizeof(int32_t), stream>>>(a);
  return cuda_status(cudaGetLastError(), "store_kvcache_fp8 launch");
}

template <typename T, int LANES>
int launch_size(const StoreArgs& a, cudaStream_t stream) {
  return a.num_tokens <= kSmallCall ? launch<T, LANES, 256, 4>(a, stream)
                                    : launch<T, LANES, 512, 4>(a, stream);
}

template <typename T>
int launch_lanes(const StoreArgs& a, cudaStream_t stream) {
  const int vectors = a.dim / 8;
  if (vectors <= 4) return launch_size<T, 4>(a, stream);
  if (vectors <= 8) return launch_size<T, 8>(a, stream);
  if (vectors <= 16) return launch_size<T, 16>(a, stream);
  return launch_size<T, 32>(a, stream);
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

extern "C" int kvoff_store_kvcache_fp8_packed(const int64_t* a) {
  if (a == nullptr) return fail(KVOFF_EINVAL, "kvoff_store_kvcache_fp8_packed: null pointer");
  return kvoff_store_kvcache_fp8(
      reinterpret_cast<const void*>(a[0]), a[1], reinterpret_cast<const void*>(a[2]), a[3],
      reinterpret_cast<void*>(a[4]), reinterpret_cast<void*>(a[5]), reinterpret_cast<float*>(a[6]),
      reinterpret_cast<float*>(a[7]), a[8], a[9], (int32_t)a[10], a[11],
      reinterpret_cast<const int32_t*>(a[12]), a[13], a[14], reinterpret_cast<int32_t*>(a[15]),
      reinterpret_cast<void*>(a[16]));
}
