// Shared by the attention kernels over the e4m3 paged cache: arguments, the
// partition of the work over CTAs, and the join of split rows.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <atomic>

#include "runtime.h"

namespace kvoff {
namespace attention {

// Keys of one step of the partition.
constexpr int kKeyTile = 128;

struct Args {
  const uint8_t* q;
  uint8_t* out;
  float* lse;  // [num_tokens, q_heads] or null
  int64_t q_stride, out_stride;  // bytes per token
  const uint8_t* cache[2];       // K, V: [pages, page, kv_heads, D]
  const float* scale[2];         // [pages, page / scale_block, kv_heads]
  const int32_t* tables;
  int64_t table_stride;
  const int32_t* contexts;
  const int32_t* starts;  // null: token s is sequence s
  float scale_log2;       // softmax scale * log2(e)
  int32_t table_width, num_pages, page, block_tiles;  // scale block in 16-key units
  int32_t page_shift;  // log2 of page, or -1 when it is no power of two
  int32_t seqs, num_tokens, q_heads, kv_heads, group;
  int32_t rows;      // packed rows of a row tile: 2^row_shift
  int32_t row_shift;
  double tiles_per_cost;  // 1 / (kKeyTile * group)
  int32_t fixed;     // what beginning and ending a row tile costs, as keys read
  int32_t max_tiles; // row tiles of the longest sequence (direct form)
  bool direct;       // one CTA per (sequence, head, row tile), nothing is split
  int32_t stride;    // CTA c works with c + stride: kv_heads when each CTA keeps to a head, else 1
  bool bf16;
  bool wide_out;     // rows of out can be written 16 bytes at a time
  uint32_t most_waits;       // of the prompt kernel: looks at a barrier before a wait gives up
  float* partial;            // 2 slots per CTA
  struct Record* records;    // one per CTA
};

// Page of a key, and the key's place in it. A division takes 30 instructions.
__device__ __forceinline__ int page_index(const Args& a, int key) {
  return a.page_shift >= 0 ? key >> a.page_shift : key / a.page;
}

// What a CTA leaves for the join: the split (sequence, head, row tile) that
// begins in it, how many CTAs after it hold parts of it, and which of its two
// slots hold a part. Slot 0 continues the previous CTA's last tile, slot 1
// begins the CTA's own last one.
struct Record {
  int32_t seq, head, tile;
  int32_t further;  // -1: none begins here
  int32_t valid[2];
  int32_t pad[2];
};

// The rows of a sequence and what they see. Row i of a (sequence, KV head) is
// query token i / group, head i % group; token t of q_len sees keys below
// context - q_len + t + 1.
struct Sequence {
  int32_t start, q_len, context, tiles;
  int64_t base;  // cost of a row tile: base + its last row's index + 1

  __device__ __forceinline__ void load(const Args& a, int s) {
    if (a.starts == nullptr) {
      start = s;
      q_len = 1;
    } else {  // kept inside q whatever the offsets say
      start = min(max(a.starts[s], 0), a.num_tokens);
      q_len = min(max(a.starts[s + 1], start), a.num_tokens) - start;
    }
    context = min(max(a.contexts[s], 0), a.table_width * a.page);  // checked to fit 32 bits
    tiles = (int32_t)(((uint32_t)(q_len * a.group) + a.rows - 1) >> a.row_shift);
    base = (int64_t)(max(context - q_len, 0) + a.fixed) * a.group;
  }
  __device__ __forceinline__ int64_t cost(const Args& a, int r) const {
    return base + min((r + 1) << a.row_shift, q_len * a.group);
  }
  // Cost of the row tiles before r (all of them whole).
  __device__ __forceinline__ int64_t before(const Args& a, int64_t r) const {
    return r * base + ((r * (r + 1) / 2) << a.row_shift);
  }
  __device__ __forceinline__ int64_t per_head(const Args& a) const {
    return tiles == 0 ? 0 : before(a, tiles - 1) + cost(a, tiles - 1);
  }
  // Keys that the last row of tile r sees.
  __device__ __forceinline__ int keys(const Args& a, int r) const {
    const int last = min((r + 1) << a.row_shift, q_len * a.group) - 1;
    return max(0, context - q_len + last / a.group + 1);
  }
};

// One row tile of one head, and the key tiles of it that a CTA works through.
struct Segment {
  int seq, head, tile;
  int begin, end, tiles;  // key tiles
  bool whole;
  int slot;  // of the partial result, when not whole
};

// Deals the work of a launch over its CTAs. With stride kv_heads, CTA c has head
// c % kv_heads, and the heads are dealt alike: CTAs that run side by side read
// the same tokens' rows of all heads, which stand next to one another in memory.
// With stride 1 the heads stand on the axis too. The key reads of all (sequence,
// head, row tile) triples, and a fixed cost of each, stand on one axis, in that
// order; each CTA takes an equal stretch of it, cut at key tiles. So a batch of unequal lengths, or one
// long sequence, keeps all SMs busy to the end, from lengths that only the
// device knows. A triple that is cut is joined by join_kernel.
//
//   Walk walk(args); while (walk.next(segment)) { ...; walk.advance(); } walk.finish() once a CTA.
template <int kThreads>
struct Walk {
  Sequence seq;
  int s, head, tile, cta;
  int64_t at, from, to, share;  // axis position of the triple; the CTA's stretch
  Record record;
  bool more;

  struct Shared {
    int64_t warp_sum[kThreads / 32];
    int64_t position;
    int32_t seq;
  };

  // Heads on this CTA's axis.
  __device__ __forceinline__ static int heads(const Args& a) { return a.stride == 1 ? a.kv_heads : 1; }

  Walk() = default;
  __device__ __forceinline__ Walk(const Args& a, Shared* sh) {
    cta = blockIdx.x;
    record.further = -1;
    record.valid[0] = record.valid[1] = 0;
    if (a.direct) {
      tile = cta % a.max_tiles;
      head = cta / a.max_tiles % a.kv_heads;
      s = cta / a.max_tiles / a.kv_heads;
      seq.load(a, s);
      more = tile < seq.tiles;
      return;
    }
    const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
    const int per = (a.seqs + kThreads - 1) / kThreads;
    const int first = min((int)threadIdx.x * per, a.seqs), last = min(first + per, a.seqs);
    int64_t mine = 0;
    for (int i = first; i < last; ++i) {
      seq.load(a, i);
      mine += heads(a) * seq.per_head(a);
    }
    int64_t sum = mine;
#pragma unroll
    for (int d = 1; d < 32; d *= 2) {
      const int64_t other = __shfl_up_sync(0xFFFFFFFFu, sum, d);
      if (lane >= d) sum += other;
    }
    if (lane == 31) sh->warp_sum[warp] = sum;
    __syncthreads();
    int64_t total = 0, before = sum - mine;
#pragma unroll
    for (int i = 0; i < kThreads / 32; ++i) {
      if (i < warp) before += sh->warp_sum[i];
      total += sh->warp_sum[i];
    }
    // A stretch of less than two key tiles costs more to join than to read.
    const int64_t least = (int64_t)(2 * kKeyTile + a.fixed) * a.group;
    const int parts = gridDim.x / a.stride;
    share = max((int64_t)((double)total / parts) + 1, least);
    from = cta / a.stride * share;
    to = min(from + share, total);
    more = from < to;
    if (more && from >= before && from < before + mine) {
      int64_t position = before;
      for (int i = first; i < last; ++i) {
        seq.load(a, i);
        const int64_t cost = heads(a) * seq.per_head(a);
        if (from < position + cost) {
          sh->position = position;
          sh->seq = i;
          break;
        }
        position += cost;
      }
    }
    __syncthreads();
    if (!more) return;
    s = sh->seq;
    at = sh->position;
    seq.load(a, s);
    const int64_t per_head = seq.per_head(a);
    if (a.stride == 1) {
      head = (int)((double)(from - at) / (double)per_head);
      while (head * per_head > from - at) --head;  // the quotient may be one off
      while ((head + 1) * per_head <= from - at) ++head;
      at += head * per_head;
    } else {
      head = cta % a.stride;
    }
    int low = 0, high = seq.tiles - 1;  // the last row tile that begins at or before `from`
    while (low < high) {
      const int mid = (low + high + 1) / 2;
      if (at + seq.before(a, mid) <= from)
        low = mid;
      else
        high = mid - 1;
    }
    tile = low;
    at += seq.before(a, tile);
  }

  // The key tile at which the axis position x cuts the current triple.
  __device__ __forceinline__ int cut(const Args& a, int64_t x, int64_t cost, int tiles) const {
    if (x >= at + cost) return tiles;
    const int64_t read = x - at - (int64_t)a.fixed * a.group;
    // In doubles: 64-bit divisions are 100 instructions, and all that counts is that
    // both sides of a cut get the same number.
    return read <= 0 ? 0 : (int)min((double)tiles, (double)read * a.tiles_per_cost);
  }

  __device__ __forceinline__ void advance(const Args& a) {
    if (a.direct) {  // more row tiles than announced: the same CTAs take them
      tile += a.max_tiles;
      more = tile < seq.tiles;
      return;
    }
    at += seq.cost(a, tile);
    more = at < to;
    if (!more || ++tile < seq.tiles) return;
    tile = 0;
    if (a.stride == 1) {
      if (++head < a.kv_heads) return;
      head = 0;
    }
    do seq.load(a, ++s);  // `to` is at most the total, so a sequence with rows follows
    while (seq.tiles == 0);
  }

  __device__ __forceinline__ bool next(const Args& a, Segment* out) {
    while (more) {
      out->seq = s;
      out->head = head;
      out->tile = tile;
      const int keys = seq.keys(a, tile);
      out->tiles = max(1, (keys + kKeyTile - 1) / kKeyTile);
      out->begin = 0;
      out->end = out->tiles;
      out->slot = 0;
      if (!a.direct) {
        const int64_t cost = seq.cost(a, tile);
        out->begin = cut(a, from, cost, out->tiles);
        out->end = cut(a, to, cost, out->tiles);
        out->slot = at >= from ? 1 : 0;
        out->whole = out->begin == 0 && out->end == out->tiles;
        const bool part = !out->whole && out->begin < out->end;
        if (part && out->slot == 0) record.valid[0] = 1;
        if (part && out->slot == 1) record.valid[1] = 1;
        if (out->slot == 1 && !out->whole) {
          record.seq = s;
          record.head = head;
          record.tile = tile;
          // The CTA in whose stretch the triple's last unit lies.
          int to_cta = cta / a.stride;
          for (int64_t end_of = to; end_of < at + cost; end_of += share) ++to_cta;
          record.further = to_cta - cta / a.stride;
        }
      } else {
        out->whole = true;
      }
      if (out->begin < out->end) return true;
      advance(a);
    }
    return false;
  }

  __device__ __forceinline__ void finish(const Args& a) const {
    if (!a.direct) a.records[cta] = record;
  }
  // Instead of it, when the work was not done: the join must not find what stood there.
  __device__ __forceinline__ void give_up(const Args& a) {
    record.further = -1;
    record.valid[0] = record.valid[1] = 0;
    finish(a);
  }
};

// A slot of the partial results: sums of p * v [rows, D], then each row's
// maximum (log2 units) and its sum of p.
__host__ __device__ inline int64_t slot_floats(int rows, int dim) {
  return (int64_t)rows * (dim + 2);
}

// Lets the join be launched while this kernel ends; it waits for the results itself.
__device__ __forceinline__ void launch_dependents() { asm volatile("griddepcontrol.launch_dependents;"); }

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// log2 of a scale of V. One that is zero is far below all others: its keys
// count in the sum of weights only. So do keys whose V is all zero.
constexpr float kZeroLog2 = -200.0f;
__device__ __forceinline__ float scale_log2_of(float scale) {
  float y;
  asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(scale));
  return scale > 0.0f ? fmaxf(y, kZeroLog2) : scale == scale ? kZeroLog2 : scale;
}

// Writes two adjacent output values of a row.
__device__ __forceinline__ void write_pair(const Args& a, int token, int q_head, int dim, int d,
                                           float x, float y) {
  uint8_t* p = a.out + token * a.out_stride + ((int64_t)q_head * dim + d) * 2;
  if (a.bf16)
    *reinterpret_cast<__nv_bfloat162*>(p) = __floats2bfloat162_rn(x, y);
  else
    *reinterpret_cast<__half2*>(p) = __floats2half2_rn(x, y);
}

__device__ __forceinline__ void write_lse(const Args& a, int token, int q_head, float m, float l) {
  // l == 0: the row sees no key.
  if (a.lse != nullptr)
    a.lse[(int64_t)token * a.q_heads + q_head] =
        l == 0.0f ? __int_as_float(0xFF800000) : (m + log2f(l)) * 0.69314718055994531f;
}

// Joins the split row tiles; one CTA of `grid` per record and 32 values of D.
int launch_join(const Args& a, int dim, int grid, cudaStream_t stream);

// The kernels. `dim` is 64 or 128; a is filled but for rows and partial.
// Rows are packed rows of a KV head: query tokens times `group`.
constexpr int kDecodeRows = 16;   // the most of one row tile; 8 when no call has more
constexpr int kExtendRows = 256;
// What beginning and ending a row tile costs, as keys read: 4 to 5 us of a decode
// step, against 0.7 us a tile of 128 keys. Without it in the partition a CTA that
// gets a hundred short sequences ends last (64 sequences of 0 to 8192 keys: 243
// us; 512 keys 47, 768 keys 46, 1024 keys 49: that batch alone was measured).
constexpr int kDecodeFixed = 768;
constexpr int kExtendFixed = 512;
// Raises a kernel's shared memory limit, once per kernel and device.
template <void (*kKernel)(Args)>
int allow_shared(int bytes) {
  static std::atomic<uint64_t> done{0};  // one for each kernel: bit d is device d
  int device = 0;
  KVOFF_TRY(cuda_status(cudaGetDevice(&device), "cudaGetDevice"));
  const uint64_t bit = device < 64 ? 1ull << device : 0;
  if ((done.load(std::memory_order_relaxed) & bit) != 0) return KVOFF_OK;
  KVOFF_TRY(cuda_status(cudaFuncSetAttribute(kKernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes),
                        "attention_fp8 shared memory"));
  done.fetch_or(bit, std::memory_order_relaxed);
  return KVOFF_OK;
}
int launch_decode(const Args& a, int dim, int grid, cudaStream_t stream);
int launch_extend(const Args& a, int dim, int grid, cudaStream_t stream);

// Error flags of extend's bounded waits on the current device.
int extend_device_error(int32_t* flags, bool clear);
constexpr int kErrExtendWaitTimeout = 2;
constexpr uint32_t kMostWaits = 1u << 20;  // looks of about a microsecond: a second in all

}  // namespace attention
}  // namespace kvoff
