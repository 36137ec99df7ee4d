// Rotary positions of q and k.
//
// A head's first R = rotary_dim values are R/2 pairs; pair j of a token at
// position p is turned by the angle p * f_j, whose cosine and sine (with the
// attention factor of a scaled rotation already in them) stand in row p of a
// table [positions, R]: cosines first, then sines.
//     y1 = x1 * c - x2 * s,   y2 = x2 * c + x1 * s
// Pair j is (x_j, x_{j + R/2}) in the half layout and (x_2j, x_2j+1) in the
// interleaved one; values from R on pass through. The transpose of the map
// (s -> -s) is its gradient. Products and sums are fp32, one rounding at the
// end.
//
// Bound by memory: each value is read and written once, and a table row is
// read once per token. A thread owns one unit of a token (the half layout: a
// 16-byte vector of the first half with its partner in the second; the
// interleaved one: a 16-byte vector, which holds whole pairs) and carries its
// cosines and sines in registers through several heads. With all heads of a
// unit in one thread a decode step of four tokens would use a few warps only,
// and with one head per thread every thread would load more table than data,
// so the heads are dealt over `lanes` threads: one head each while there are
// fewer threads of four heads than 2048 an SM, four from there on. The values are loaded
// before the position is known, so one latency and not three stands between
// them and the result.
//
// Measured: 16384 tokens, 64 + 8 heads of 128 bf16 in 93 us = 6.6 TB/s, a
// copy's rate (197 us with the table row waited for first and two-byte
// accesses to registers); 4096 tokens, 32 + 8 heads in 15.4 us; 4 tokens in
// 2.2 us. Five heads a thread spill (30 us for the 4096 tokens), eight leave
// too few threads (22 us). 80 registers leave 768 threads an SM, so with one
// head a thread the sizes below that border run in several rounds: 500 tokens
// 3.7 us, 1000 5.4, 2000 9.0, 3500 17.1, where the bytes take 1.6, 3.2, 6.4 and 11.2.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "runtime.h"

namespace kvoff {
namespace {

constexpr int kThreads = 256;
constexpr int kUnroll = 4;  // heads whose loads are in flight at once

struct RotaryArgs {
  const uint8_t* in[2];  // q, k
  uint8_t* out[2];
  int64_t in_stride[2], out_stride[2];  // bytes per token
  const void* positions;
  const float* table;
  int64_t table_rows, num_tokens;
  int32_t* bad_positions;
  int32_t heads[2];
  int32_t dim, rotary_dim;
  int32_t units, turning;  // units of a head; the first `turning` hold pairs
  int32_t lanes, tokens_per_cta;
  float sign;       // of the sines: -1 for the transpose
  bool positions64, copy;  // copy: units that pass through are written too
  bool wide_table;         // its rows' halves can be read 16 bytes at a time
};

// V adjacent values of a row as they stand in memory, read and written as 32-bit
// words where there is a whole one.
template <typename T, int V>
struct Vec {
  static constexpr int kBytes = sizeof(T) * V;
  uint32_t w[kBytes < 4 ? 1 : kBytes / 4];

  __device__ __forceinline__ void load(const uint8_t* p) {
    if constexpr (kBytes == 16) {
      const uint4 v = *reinterpret_cast<const uint4*>(p);
      w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
    } else if constexpr (kBytes == 8) {
      const uint2 v = *reinterpret_cast<const uint2*>(p);
      w[0] = v.x, w[1] = v.y;
    } else if constexpr (kBytes == 4) {
      w[0] = *reinterpret_cast<const uint32_t*>(p);
    } else {
      w[0] = *reinterpret_cast<const uint16_t*>(p);
    }
  }
  __device__ __forceinline__ void store(uint8_t* p) const {
    if constexpr (kBytes == 16)
      *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
    else if constexpr (kBytes == 8)
      *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
    else if constexpr (kBytes == 4)
      *reinterpret_cast<uint32_t*>(p) = w[0];
    else
      *reinterpret_cast<uint16_t*>(p) = (uint16_t)w[0];
  }
  __device__ __forceinline__ void unpack(float (&x)[V]) const {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < V; ++i) x[i] = __uint_as_float(w[i]);
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const uint32_t u = w[i / 2];
        if constexpr (std::is_same<T, __half>::value)
          x[i] = __half2float(__ushort_as_half((unsigned short)(i % 2 ? u >> 16 : u & 0xFFFFu)));
        else
          x[i] = __uint_as_float(i % 2 ? u & 0xFFFF0000u : u << 16);
      }
    }
  }
  __device__ __forceinline__ void pack(const float (&x)[V]) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < V; ++i) w[i] = __float_as_uint(x[i]);
    } else {
#pragma unroll
      for (int i = 0; i < V; i += 2) {
        const float low = x[i], high = V > 1 ? x[(i + 1) % V] : 0.0f;
        if constexpr (std::is_same<T, __half>::value)
          asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(w[i / 2]) : "f"(high), "f"(low));
        else
          asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(w[i / 2]) : "f"(high), "f"(low));
      }
    }
  }
};

// V values per vector; a unit is two vectors in the half layout, one else.
template <typename T, int V, bool kInterleaved>
__global__ void __launch_bounds__(kThreads, 3)
    rotary_kernel(const __grid_constant__ RotaryArgs a) {
  constexpr int kPairs = kInterleaved ? V / 2 : V;
  using Vector = Vec<T, V>;
  const int per_token = a.units * a.lanes;
  const int64_t token = (int64_t)blockIdx.x * a.tokens_per_cta + threadIdx.x / per_token;
  const int rest = threadIdx.x % per_token;
  const int unit = rest % a.units, lane = rest / a.units;
  if (threadIdx.x >= a.tokens_per_cta * per_token || token >= a.num_tokens) return;
  const bool turns = unit < a.turning;
  if (!turns && !a.copy) return;
  const int half = a.rotary_dim / 2;
  // First value of the unit, and of its partner vector.
  const int at = turns ? unit * V : a.rotary_dim + (unit - a.turning) * V;
  const int partner = (!kInterleaved && turns) ? half : 0;
  const int heads = a.heads[0] + a.heads[1];
  const int row = a.dim * (int)sizeof(T);
  const uint8_t* in_q = a.in[0] + token * a.in_stride[0] + at * sizeof(T);
  const uint8_t* in_k = a.in[1] + token * a.in_stride[1] + at * sizeof(T) - a.heads[0] * row;
  uint8_t* out_q = a.out[0] + token * a.out_stride[0] + at * sizeof(T);
  uint8_t* out_k = a.out[1] + token * a.out_stride[1] + at * sizeof(T) - a.heads[0] * row;

  const int64_t position = a.positions64 ? __ldg(static_cast<const long long*>(a.positions) + token)
                                         : __ldg(static_cast<const int32_t*>(a.positions) + token);
  // The first heads' values are on the way while the table row is looked up.
  Vector x[kUnroll], y[kUnroll];
  auto load = [&](int first) {
#pragma unroll
    for (int i = 0; i < kUnroll; ++i) {
      const int h = first + i * a.lanes;
      if (h < heads) {
        const uint8_t* p = (h < a.heads[0] ? in_q : in_k) + h * row;
        x[i].load(p);
        if (!kInterleaved) y[i].load(p + partner * sizeof(T));
      }
    }
  };
  load(lane);
  if (position < 0) return;
  if (position >= a.table_rows) {
    if (rest == 0 && a.bad_positions != nullptr) atomicAdd(a.bad_positions, 1);
    return;
  }
  float c[kPairs], s[kPairs];
  if (turns) {
    const float* from = a.table + position * a.rotary_dim + unit * kPairs;
    constexpr int kWide = kPairs % 4 == 0 ? 4 : 1;
#pragma unroll
    for (int i = 0; i < kPairs; i += kWide) {
      if (kWide == 4 && a.wide_table) {
        const float4 u = __ldg(reinterpret_cast<const float4*>(from + i));
        const float4 v = __ldg(reinterpret_cast<const float4*>(from + half + i));
        c[i] = u.x, c[i + kWide / 4] = u.y, c[i + kWide / 2] = u.z, c[i + kWide * 3 / 4] = u.w;
        s[i] = v.x, s[i + kWide / 4] = v.y, s[i + kWide / 2] = v.z, s[i + kWide * 3 / 4] = v.w;
      } else {
#pragma unroll
        for (int j = 0; j < kWide; ++j) c[i + j] = __ldg(from + i + j), s[i + j] = __ldg(from + half + i + j);
      }
    }
#pragma unroll
    for (int i = 0; i < kPairs; ++i) s[i] *= a.sign;
  }
  for (int first = lane; first < heads; first += kUnroll * a.lanes) {
    if (first != lane) load(first);
#pragma unroll
    for (int i = 0; i < kUnroll; ++i) {
      const int h = first + i * a.lanes;
      if (h < heads) {
        uint8_t* p = (h < a.heads[0] ? out_q : out_k) + h * row;
        if (turns) {
          float u[V], v[V];
          x[i].unpack(u);
          if (kInterleaved) {
#pragma unroll
            for (int j = 0; j < kPairs; ++j) {
              const float x1 = u[2 * j], x2 = u[2 * j + 1];
              u[2 * j] = x1 * c[j] - x2 * s[j];
              u[2 * j + 1] = x2 * c[j] + x1 * s[j];
            }
          } else {
            y[i].unpack(v);
#pragma unroll
            for (int j = 0; j < kPairs; ++j) {
              const float x1 = u[j], x2 = v[j];
              u[j] = x1 * c[j] - x2 * s[j];
              v[j] = x2 * c[j] + x1 * s[j];
            }
            y[i].pack(v);
            y[i].store(p + partner * sizeof(T));
          }
          x[i].pack(u);
        }
        x[i].store(p);
      }
    }
  }
}

template <typename T, int V, bool kInterleaved>
int launch(RotaryArgs a, cudaStream_t stream) {
  a.turning = a.rotary_dim / (kInterleaved ? V : 2 * V);
  a.units = a.turning + (a.copy ? (a.dim - a.rotary_dim) / V : 0);
  const int heads = a.heads[0] + a.heads[1];
  if (a.units > kThreads)
    return fail(KVOFF_EINVAL, "kvoff_rotary: heads of %d values at this alignment are not supported",
                a.dim);
  // Four heads a thread once the threads of four heads are 2048 an SM (2.7 times
  // what is resident); below that, as many lanes as the block has room for. Only
  // 4, 1023, 4096 and 16384 tokens were measured when the border was set.
  const int64_t full = (int64_t)sm_count() * 2048;
  int lanes = (heads + kUnroll - 1) / kUnroll;
  if (a.num_tokens * a.units * lanes < full) lanes = heads;
  const int most = kThreads / a.units;
  a.lanes = lanes < most ? lanes : most;
  const int per_token = a.units * a.lanes;
  a.tokens_per_cta = a.num_tokens * per_token < full ? 1 : kThreads / per_token;
  const int threads = (a.tokens_per_cta * per_token + 31) / 32 * 32;
  const int64_t grid = (a.num_tokens + a.tokens_per_cta - 1) / a.tokens_per_cta;
  rotary_kernel<T, V, kInterleaved><<<(unsigned)grid, threads, 0, stream>>>(a);
  return cuda_status(cudaGetLastError(), "rotary launch");
}

template <typename T>
int launch_layout(const RotaryArgs& a, bool interleaved, uintptr_t bits, cudaStream_t stream) {
  constexpr int V = 16 / sizeof(T);
  // The vector forms need every address and stride in whole vectors, and a
  // rotated part (per half, in the half layout) of whole vectors.
  const bool wide = (bits & 15u) == 0 && a.dim % V == 0;
  if (interleaved)
    return wide && a.rotary_dim % V == 0 ? launch<T, V, true>(a, stream)
                                         : launch<T, 2, true>(a, stream);
  return wide && a.rotary_dim % (2 * V) == 0 ? launch<T, V, false>(a, stream)
                                             : launch<T, 1, false>(a, stream);
}

}  // namespace
}  // namespace kvoff

using namespace kvoff;

extern "C" int kvoff_rotary(const void* q, int64_t q_stride_bytes, void* q_out,
                            int64_t q_out_stride_bytes, int64_t q_heads, const void* k,
                            int64_t k_stride_bytes, void* k_out, int64_t k_out_stride_bytes,
                            int64_t kv_heads, int64_t head_dim, int64_t rotary_dim, int32_t dtype,
                            const void* positions, int32_t position_bytes, const float* table,
                            int64_t table_rows, int64_t num_tokens, int32_t flags,
                            int32_t* bad_positions, void* stream) {
  if (injected("rotary")) return KVOFF_EINJECTED;
  if (num_tokens < 0 || q_heads < 0 || kv_heads < 0 || q_heads + kv_heads <= 0 || head_dim <= 0 ||
      table_rows < 0 || q_stride_bytes < 0 || q_out_stride_bytes < 0 || k_stride_bytes < 0 ||
      k_out_stride_bytes < 0 || q_heads + kv_heads > 65535 || head_dim > 65535)
    return fail(KVOFF_EINVAL, "kvoff_rotary: bad sizes");
  if (rotary_dim <= 0 || rotary_dim % 2 != 0 || rotary_dim > head_dim)
    return fail(KVOFF_EINVAL, "kvoff_rotary: rotary_dim %lld must be even and at most head_dim %lld",
                (long long)rotary_dim, (long long)head_dim);
  if (dtype != KVOFF_BF16 && dtype != KVOFF_FP16 && dtype != KVOFF_FP32)
    return fail(KVOFF_EINVAL, "kvoff_rotary: unknown dtype %d", (int)dtype);
  if (position_bytes != 4 && position_bytes != 8)
    return fail(KVOFF_EINVAL, "kvoff_rotary: positions are int32 or int64");
  if ((flags & ~(KVOFF_ROTARY_INTERLEAVED | KVOFF_ROTARY_INVERSE)) != 0)
    return fail(KVOFF_EINVAL, "kvoff_rotary: unknown flags %d", (int)flags);
  if ((q_heads + kv_heads) * head_dim > 0x1FFFFFFFll)
    return fail(KVOFF_EINVAL, "kvoff_rotary: a token's heads exceed 2 GB");
  if (num_tokens == 0) return ok();
  if (num_tokens > 0x7FFFFFFFll)
    return fail(KVOFF_EINVAL, "kvoff_rotary: %lld tokens exceed one launch",
                (long long)num_tokens);
  if ((q_heads > 0 && (q == nullptr || q_out == nullptr)) ||
      (kv_heads > 0 && (k == nullptr || k_out == nullptr)) || positions == nullptr ||
      table == nullptr)
    return fail(KVOFF_EINVAL, "kvoff_rotary: null pointer");
  const bool interleaved = (flags & KVOFF_ROTARY_INTERLEAVED) != 0;
  const int elem = dtype == KVOFF_FP32 ? 4 : 2;
  uintptr_t bits = 0;
  if (q_heads > 0)
    bits |= reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(q_out) |
            (uintptr_t)q_stride_bytes | (uintptr_t)q_out_stride_bytes;
  if (kv_heads > 0)
    bits |= reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(k_out) |
            (uintptr_t)k_stride_bytes | (uintptr_t)k_out_stride_bytes;
  // The narrow interleaved form moves one pair at a time.
  const int narrow = interleaved ? 2 * elem : elem;
  if (bits % narrow != 0 || (interleaved && head_dim % 2 != 0))
    return fail(KVOFF_EINVAL, "kvoff_rotary: rows must be aligned to %d bytes%s", narrow,
                interleaved ? " and hold an even number of values" : "");
  // Rows written on top of one another, or over rows that are still to be read.
  if (num_tokens > 1 &&
      ((q_heads > 0 && q_out_stride_bytes < q_heads * head_dim * elem) ||
       (kv_heads > 0 && k_out_stride_bytes < kv_heads * head_dim * elem)))
    return fail(KVOFF_EINVAL, "kvoff_rotary: rows of the output overlap");
  if (num_tokens > 1 && ((q_heads > 0 && q == q_out && q_stride_bytes != q_out_stride_bytes) ||
                         (kv_heads > 0 && k == k_out && k_stride_bytes != k_out_stride_bytes)))
    return fail(KVOFF_EINVAL, "kvoff_rotary: in place the strides of input and output are equal");
  RotaryArgs a{};
  a.in[0] = static_cast<const uint8_t*>(q);
  a.in[1] = static_cast<const uint8_t*>(k);
  a.out[0] = static_cast<uint8_t*>(q_out);
  a.out[1] = static_cast<uint8_t*>(k_out);
  a.in_stride[0] = q_stride_bytes;
  a.in_stride[1] = k_stride_bytes;
  a.out_stride[0] = q_out_stride_bytes;
  a.out_stride[1] = k_out_stride_bytes;
  a.positions = positions;
  a.positions64 = position_bytes == 8;
  a.table = table;
  a.table_rows = table_rows;
  a.num_tokens = num_tokens;
  a.bad_positions = bad_positions;
  a.heads[0] = (int32_t)q_heads;
  a.heads[1] = (int32_t)kv_heads;
  a.dim = (int32_t)head_dim;
  a.rotary_dim = (int32_t)rotary_dim;
  a.sign = (flags & KVOFF_ROTARY_INVERSE) != 0 ? -1.0f : 1.0f;
  a.wide_table = rotary_dim % 8 == 0 && (reinterpret_cast<uintptr_t>(table) & 15u) == 0;
  a.copy = rotary_dim < head_dim &&
           ((q_heads > 0 && q != q_out) || (kv_heads > 0 && k != k_out));
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  int rc;
  if (dtype == KVOFF_BF16)
    rc = launch_layout<__nv_bfloat16>(a, interleaved, bits, s);
  else if (dtype == KVOFF_FP16)
    rc = launch_layout<__half>(a, interleaved, bits, s);
  else
    rc = launch_layout<float>(a, interleaved, bits, s);
  if (rc != KVOFF_OK) return rc;
  return ok();
}

extern "C" int kvoff_rotary_packed(const int64_t* a) {
  if (a == nullptr) return fail(KVOFF_EINVAL, "kvoff_rotary_packed: null pointer");
  return kvoff_rotary(reinterpret_cast<const void*>(a[0]), a[1], reinterpret_cast<void*>(a[2]), a[3],
                      a[4], reinterpret_cast<const void*>(a[5]), a[6], reinterpret_cast<void*>(a[7]),
                      a[8], a[9], a[10], a[11], (int32_t)a[12], reinterpret_cast<const void*>(a[13]),
                      (int32_t)a[14], reinterpret_cast<const float*>(a[15]), a[16], a[17],
                      (int32_t)a[18], reinterpret_cast<int32_t*>(a[19]),
                      reinterpret_cast<void*>(a[20]));
}
