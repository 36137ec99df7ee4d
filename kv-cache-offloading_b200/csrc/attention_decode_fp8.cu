// Attention of a few query rows over the e4m3 paged cache: decode steps, and
// any row count that does not fill a 128-row tensor tile.
//
//     o_i = sum_t p_it v_t / sum_t p_it,  p_it = exp(c q_i . k_t - m_i)
//
// Bound by the cache's bytes: with `group` query heads a KV head a key costs
// 2 D bytes and 4 D group flops. The kernel therefore reads every byte once,
// keeps about 160 KB of loads in flight on each SM, and spends as few
// instructions a byte as it can. Measured: 4 sequences of 34816 keys, 32 / 8
// heads of 128, in 60 us = 4.8 TB/s, 0.73 of a copy's rate; from 34816 to 69632
// keys it adds 45 us, so about 15 us of it begin and end the call (the walk
// over the lengths 1.8, first addresses 1.9, first tiles 1.5, the join of the
// warps 1.3, the join kernel 2.3 us, the launches).
//
// * A warp works alone on 16-key tiles: its own ring of kStages tiles of K
//   and V in shared memory, filled by cp.async, 4 KB a tile at D = 128. No
//   barrier of the CTA is waited for until the end of a segment. While the warps
//   are joined there, the next segment's first tiles and its q are on their way
//   (64 sequences of up to 8192 keys: 46.4 us; 1.3 more without).
// * Scores: S^T[16 keys, 8 rows] = K Q^T by mma.m16n8k16 in f16. K is the M
//   operand, so the 8 columns are the query rows of one KV head (group 4 fills
//   half of them, group 8 all). e4m3 is a subset of f16, so K is exact; q is
//   scaled by a power of two to an amax of 2^14..2^15, where every bf16 value
//   down to 2^-31 of the row's largest and every f16 value is exact too. The
//   D axis is permuted (the same way for K and Q), so that each thread's
//   fragment of K is 16 contiguous bytes.
// * O^T[D, 8 rows] += V^T P^T, with V^T the M operand: pairs of keys are
//   brought together byte by byte (prmt) and converted like K; P goes from the
//   accumulator layout to the operand's by movmatrix. The scale of V is one
//   number for the tile (a scale block is 16 tokens or more) and is put into
//   P = 2^(x - m) scale / 2^t, where 2^(m + t + 8) follows the largest 2^x scale
//   that the row itself has met: f16 holds terms down to 2^-22 of the row's
//   largest one at full precision, whatever scales other rows' keys have, or
//   keys of no weight. Keys whose V is all zero do not count there: beside a
//   large value, seen or not, a scale block holds little else. The sum of
//   2^(x - m) does not depend on t.
// * m and t are raised only when a score, or a score with its scale, passes
//   them by more than 2^6 (one vote a tile, on the lower of the two limits); until
//   then P is at most 2^14 in f16. Rescaling is rare then, and the reductions over
//   keys stay out of the loop.
//
// Masked scores are -inf before anything depends on them. Rows of K and V
// behind the context are not read (cp.async fills zeros), since 0 * NaN would
// not be 0; where a tile is hidden from some rows and seen by others, NaN
// values of V take a separate path (see nan_tile).
#include "attention_fp8.h"
#include "codec.cuh"

namespace kvoff {
namespace attention {
namespace {

constexpr int kWarps = 8;
constexpr int kThreads = 32 * kWarps;
constexpr int kTile = 16;           // keys of a warp's tile
constexpr float kRaise = 6.0f;      // log2 of how far P may pass 1
constexpr float kWeightLog2 = 8.0f; // of the largest P in f16
constexpr float kLeastUnit = -126.0f;  // of t
constexpr uint32_t kNegInf = 0xFF800000u;
static_assert(kKeyTile == kWarps * kTile, "one tile a warp and key tile");

// One CTA an SM, eight warps with all the registers they can use. With two CTAs
// at 128 registers (and half the stages each) 16 rows were spilled (138 us, now
// 77: 4 x 34816 keys, 8 heads of 128, 12 rows) and 8 rows took 69 us, now 60. Two
// tiles in one step take as long as one (60).
template <int D, int NT>
struct Shape {
  static constexpr int kTileBytes = kTile * D;             // of K, and of V
  static constexpr int kStageBytes = 2 * kTileBytes + 16;  // and the two scales
  static constexpr int kStages = D == 64 ? 8 : 6;
  static constexpr int kWarpBytes = kStages * kStageBytes;
  // A warp's sums at the end of a segment take its last stages; the others hold the
  // next segment's first tiles by then.
  static constexpr int kPitch = D + 4;
  static constexpr int kSumsBytes = 8 * NT * kPitch * 4;
  static constexpr int kEarly = kStages - (kSumsBytes + kStageBytes - 1) / kStageBytes;
  static constexpr int kSumsAt = kEarly * kStageBytes;
  static constexpr int kQueryBytes = 8 * NT * D * 2;  // q of a row tile, as it stands in memory
  static constexpr int kBytes = kWarps * kWarpBytes + 2 * kQueryBytes;
  static_assert(kEarly > 0 && kEarly < kStages && kStageBytes % 16 == 0, "stages");
};

__device__ __forceinline__ uint32_t smem_of(const void* p) {
  return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}

template <int kBytes>
__device__ __forceinline__ void copy_async(uint32_t dst, const void* src) {
  if (kBytes == 16)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
  else
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}
// 16 bytes, or zeros without a look at src.
__device__ __forceinline__ void copy_async_or_zero(uint32_t dst, const void* src, bool real) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(real ? 16 : 0)
               : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

__device__ __forceinline__ uint4 load_shared16(uint32_t p) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "r"(p)
               : "memory");
  return v;
}
__device__ __forceinline__ uint2 load_shared8(uint32_t p) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(p) : "memory");
  return v;
}
__device__ __forceinline__ float2 load_shared_f2(uint32_t p) {
  float2 v;
  asm volatile("ld.shared.v2.f32 {%0,%1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(p) : "memory");
  return v;
}

// Two e4m3 (low or high half of w) -> f16x2, exact.
__device__ __forceinline__ uint32_t widen_low(uint32_t w) {
  uint32_t r;
  asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, l;\n\t}" : "=r"(r) : "r"(w));
  return r;
}
__device__ __forceinline__ uint32_t widen_high(uint32_t w) {
  uint32_t r;
  asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, h;\n\t}" : "=r"(r) : "r"(w));
  return r;
}

__device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                    uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

__device__ __forceinline__ uint32_t pack_half(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

// Where 16-byte chunk `chunk` of row `row` of a K or V tile stands, so that a
// warp's fragment reads meet no bank twice. K is read as (8 rows) x (4 chunks
// side by side), V as every other row at one 16-byte (D = 64: 8-byte) column.
template <int D>
__device__ __forceinline__ uint32_t k_place(int row, int chunk) {
  return D == 128 ? row * D + ((chunk ^ (row & 1) * 4) * 16) : row * D + chunk * 16;
}
template <int D>
__device__ __forceinline__ uint32_t v_place(int row, int chunk) {
  if (D == 128) return row * D + ((chunk ^ ((row >> 1) & 3) * 2) * 16);
  return (row ^ ((row >> 2) & 1)) * D + ((chunk ^ ((row >> 1) & 1) * 2) * 16);
}

// The values of V that one thread feeds to the M = D operand of a 16-key
// tile: bytes d0 .. d0 + D/8 of keys 2t, 2t+1, 2t+8, 2t+9.
template <int D>
struct VTile {
  static constexpr int kWords = D / 32;
  uint32_t w[4][kWords];

  __device__ __forceinline__ void load(uint32_t tile, int g, int t) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int row = 2 * t + (i & 1) + (i >> 1) * 8;
      if (D == 128) {
        const uint4 v = load_shared16(tile + v_place<D>(row, g));
        w[i][0] = v.x, w[i][1] = v.y, w[i][kWords - 2] = v.z, w[i][kWords - 1] = v.w;
      } else {
        const uint2 v = load_shared8(tile + v_place<D>(row, g / 2) + (g & 1) * 8);
        w[i][0] = v.x, w[i][1] = v.y;
      }
    }
  }
  // The tile's keys with a value that is not zero, one bit each. All lanes of the warp call it.
  __device__ __forceinline__ uint32_t filled() const {
    uint32_t keys = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint32_t any = 0;
#pragma unroll
      for (int k = 0; k < kWords; ++k) any |= w[i][k];
      uint32_t lanes = __ballot_sync(0xFFFFFFFFu, (any & 0x7F7F7F7Fu) != 0);
      lanes |= lanes >> 16;
      lanes |= lanes >> 8;
      lanes |= lanes >> 4;  // bit t: key 2t + (i & 1) + 8 (i >> 1)
#pragma unroll
      for (int t = 0; t < 4; ++t) keys |= (lanes >> t & 1) << (2 * t + (i & 1) + (i >> 1) * 8);
    }
    return keys;
  }
  // Fragment of M tile i (values d0 + 2i in rows g, d0 + 2i + 1 in rows g + 8).
  __device__ __forceinline__ void fragment(int i, uint32_t (&a)[4]) const {
    const uint32_t pick = (i & 1) ? 0x7362 : 0x5140;  // bytes 2, 3 or 0, 1 of both keys
    const uint32_t low = __byte_perm(w[0][i / 2], w[1][i / 2], pick);
    const uint32_t high = __byte_perm(w[2][i / 2], w[3][i / 2], pick);
    a[0] = widen_low(low), a[1] = widen_high(low);
    a[2] = widen_low(high), a[3] = widen_high(high);
  }
};

// The largest of a column's values, over the lanes that hold its keys.
__device__ __forceinline__ float column_most(float x) {
  x = fmaxf(x, __shfl_xor_sync(0xFFFFFFFFu, x, 4));
  x = fmaxf(x, __shfl_xor_sync(0xFFFFFFFFu, x, 8));
  return fmaxf(x, __shfl_xor_sync(0xFFFFFFFFu, x, 16));
}

// scale / 2^t. What passes 2^126 is put into the scores, see kMostWeight.
constexpr float kMostWeight = 126.0f;
__device__ __forceinline__ float weight_of(float x) { return exp2_fast(x > kMostWeight ? kMostWeight : x); }

// One warp's state over a segment.
template <int D, int NT>
struct Rows {
  static constexpr int kSteps = D / 16;
  uint32_t q[NT][kSteps][2];  // operand fragments of the scaled q
  float factor[NT][2];        // log2 units of a raw score, columns 2t and 2t+1
  int limit[NT][2];           // keys that the column's row sees
  float o[kSteps][NT][4];
  float m[NT][2], l[NT][2];   // l: sum of 2^(x - m)
  float unit[NT][2];          // t: o is the sum of 2^(x - m - t) v
  float far;                  // log2 of the largest V scale that is no more than 2^kMostWeight units of any row
};

template <int D, int NT>
__device__ __forceinline__ void load_rows(const Args& a, const Sequence& seq, const Segment& seg,
                                          uint32_t queries, int g, int t, Rows<D, NT>& r) {
  const int total = seq.q_len * a.group;
#pragma unroll
  for (int j = 0; j < NT; ++j) {
    const int row = seg.tile * a.rows + 8 * j + g;
    const bool real = row < total;
    uint4 raw[D / 64][2];
    uint32_t amax = 0;
    if (real) {
      const uint32_t p = queries + (8 * j + g) * D * 2;
#pragma unroll
      for (int c = 0; c < D / 64; ++c)
#pragma unroll
        for (int i = 0; i < 2; ++i) raw[c][i] = load_shared16(p + (64 * c + 16 * t + 8 * i) * 2);
    } else {
#pragma unroll
      for (int c = 0; c < D / 64; ++c) raw[c][0] = raw[c][1] = make_uint4(0, 0, 0, 0);
    }
    float x[D / 4];
#pragma unroll
    for (int c = 0; c < D / 64; ++c)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const uint32_t w[4] = {raw[c][i].x, raw[c][i].y, raw[c][i].z, raw[c][i].w};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          float2 f;
          if (a.bf16)
            f = make_float2(__uint_as_float(w[k] << 16), __uint_as_float(w[k] & 0xFFFF0000u));
          else
            f = __half22float2(*reinterpret_cast<const __half2*>(&w[k]));
          x[16 * c + 8 * i + 2 * k] = f.x;
          x[16 * c + 8 * i + 2 * k + 1] = f.y;
        }
      }
#pragma unroll
    for (int i = 0; i < D / 4; ++i) {
      const uint32_t u = __float_as_uint(x[i]) & 0x7FFFFFFFu;
      if (u < 0x7F800000u) amax = max(amax, u);
    }
    amax = max(amax, __shfl_xor_sync(0xFFFFFFFFu, amax, 1));
    amax = max(amax, __shfl_xor_sync(0xFFFFFFFFu, amax, 2));
    // 2^e with amax * 2^e in [2^14, 2^15); both it and its inverse are normal.
    const int e = amax == 0 ? 0 : min(14 - ((int)(amax >> 23) - 127), 100);
    const float up = __uint_as_float((uint32_t)(127 + e) << 23);
    const float down = a.scale_log2 * __uint_as_float((uint32_t)(127 - e) << 23);
#pragma unroll
    for (int c = 0; c < D / 64; ++c)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        r.q[j][4 * c + i][0] = pack_half(x[16 * c + 4 * i] * up, x[16 * c + 4 * i + 1] * up);
        r.q[j][4 * c + i][1] = pack_half(x[16 * c + 4 * i + 2] * up, x[16 * c + 4 * i + 3] * up);
      }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int column = 2 * t + i;
      r.factor[j][i] = __shfl_sync(0xFFFFFFFFu, down, column * 4);
      const int at = seg.tile * a.rows + 8 * j + column;
      r.limit[j][i] = at < total ? max(0, seq.context - seq.q_len + at / a.group + 1) : 0;
      r.m[j][i] = __uint_as_float(kNegInf);
      r.l[j][i] = 0.0f;
      r.unit[j][i] = kLeastUnit;
    }
  }
  r.far = 1e30f;
#pragma unroll
  for (int i = 0; i < Rows<D, NT>::kSteps; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int k = 0; k < 4; ++k) r.o[i][j][k] = 0.0f;
}

// O += V^T P^T of a tile where some of V is NaN and some rows do not see all
// keys: V's NaN are left out of the product, and a second product of their
// places with the keys that each row sees says which sums they make NaN.
template <int D, int NT>
__device__ __forceinline__ void nan_tile(const VTile<D>& v, const uint32_t (&p)[NT][2],
                                      const uint32_t (&seen)[NT][2], Rows<D, NT>& r) {
#pragma unroll
  for (int i = 0; i < D / 16; ++i) {
    uint32_t a[4], clean[4], places[4];
    v.fragment(i, a);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const uint32_t lo = (a[k] & 0x7FFFu) > 0x7C00u, hi = (a[k] >> 16 & 0x7FFFu) > 0x7C00u;
      clean[k] = (lo ? 0 : a[k] & 0xFFFFu) | (hi ? 0 : a[k] & 0xFFFF0000u);
      places[k] = (lo ? 0x3C00u : 0) | (hi ? 0x3C000000u : 0);
    }
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      mma(r.o[i][j], clean[0], clean[1], clean[2], clean[3], p[j][0], p[j][1]);
      float hit[4] = {0.0f, 0.0f, 0.0f, 0.0f};
      mma(hit, places[0], places[1], places[2], places[3], seen[j][0], seen[j][1]);
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (hit[k] > 0.0f) r.o[i][j][k] = __uint_as_float(0x7FC00000u);
    }
  }
}

template <int D, int NT>
__global__ void __launch_bounds__(kThreads, 1) attention_decode_fp8_kernel(const __grid_constant__ Args a) {
  using S = Shape<D, NT>;
  constexpr int kSteps = D / 16;
  constexpr int kRows = 8 * NT;
  extern __shared__ __align__(128) uint8_t shared[];
  __shared__ typename Walk<kThreads>::Shared walk_shared;
  __shared__ float warp_m[kWarps][kRows], warp_l[kWarps][kRows];
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, g = lane / 4, t = lane % 4;
  const uint32_t ring = smem_of(shared) + warp * S::kWarpBytes;
  const int page_tiles = a.page / kTile;
  const int64_t row_bytes = (int64_t)a.kv_heads * D;

  const int blocks = page_tiles / a.block_tiles;  // scale blocks of a page
  // This lane's 16-byte chunk of rows row0, row0 + kRowStep, ... of a tile.
  constexpr int kRowStep = 32 / (D / 16), kCopies = kTile / kRowStep;
  const int row0 = lane / (D / 16), chunk0 = lane % (D / 16);

  Walk<kThreads> walk(a, &walk_shared);
  Segment seg, coming;
  bool more = walk.next(a, &seg);
  if (more) {
    Sequence seq = walk.seq;
    auto keys_of = [&](const Segment& of, const Sequence& in) {
      return min(in.keys(a, of.tile), in.context);
    };
    // q of a segment's rows, on its way to one of two places in shared memory.
    auto fetch_queries = [&](const Segment& of, const Sequence& in, uint32_t to) {
      const int at = of.tile * a.rows + threadIdx.x / (D / 8);
      if (threadIdx.x < kRows * D / 8 && at < in.q_len * a.group) {
        const int token = in.start + at / a.group, head = of.head * a.group + at % a.group;
        copy_async<16>(to + threadIdx.x * 16,
                       a.q + token * a.q_stride + ((int64_t)head * D + threadIdx.x % (D / 8) * 8) * 2);
      }
    };
    // Where a segment's tiles of this warp stand, 32 at a time: lane l has the page
    // of tile i + l (-1: none) until it is needed, then the tile's first byte in the
    // cache (negative: no page) and its scale's index. The divisions are made once
    // for each tile here, not by every lane in the loop.
    auto page_of = [&](const Segment& of, int keys, int i) {
      const int tile = (of.begin + i + lane) * kWarps + warp;
      return i + lane < of.end - of.begin && tile * kTile < keys
                 ? __ldg(a.tables + of.seq * a.table_stride + tile / page_tiles) : -1;
    };
    int64_t place;
    int32_t block = 0;
    auto look_up = [&](const Segment& of, int i, int id) {
      const int tile = (of.begin + i + lane) * kWarps + warp, in_page = tile % page_tiles;
      place = -1;
      if (id >= 0 && id < a.num_pages) {
        place = ((int64_t)id * a.page + in_page * kTile) * row_bytes;
        block = id * blocks + in_page / a.block_tiles;
      }
    };
    uint32_t queries = smem_of(shared) + kWarps * S::kWarpBytes;  // of this segment
    const uint32_t both = 2 * queries + S::kQueryBytes;           // this segment's place and the next one's
    fetch_queries(seg, seq, queries);
    copy_commit();
    int keys = keys_of(seg, seq);  // that any row sees
    int page_next = -1, page_coming = -1;
    look_up(seg, 0, page_of(seg, keys, 0));
    uint32_t absent = 0;  // bit k: the tile issued k tiles ago has no page

    auto issue = [&](int i, int slot) {
      if (i < seg.end - seg.begin) {
        if (i > 0 && i % 32 == 0) look_up(seg, i, page_next);
        if (i % 32 == 8) page_next = page_of(seg, keys, i - 8 + 32);
        const int64_t at = __shfl_sync(0xFFFFFFFFu, place, i % 32);
        const int32_t scale = __shfl_sync(0xFFFFFFFFu, block, i % 32);
        const int left = keys - ((seg.begin + i) * kWarps + warp) * kTile;  // keys of the tile that are read
        absent = absent << 1 | (at < 0 ? 1u : 0u);
        const uint32_t stage = ring + slot * S::kStageBytes;
        const int64_t mine = at + row0 * row_bytes + seg.head * D + chunk0 * 16;
        const uint8_t* k = a.cache[0] + mine;
        const uint8_t* v = a.cache[1] + mine;
        if (at >= 0 && left >= kTile) {
#pragma unroll
          for (int c = 0; c < kCopies; ++c) {
            copy_async<16>(stage + k_place<D>(row0 + kRowStep * c, chunk0), k);
            copy_async<16>(stage + S::kTileBytes + v_place<D>(row0 + kRowStep * c, chunk0), v);
            k += kRowStep * row_bytes;
            v += kRowStep * row_bytes;
          }
        } else if (at >= 0) {
#pragma unroll
          for (int c = 0; c < kCopies; ++c) {
            const bool real = row0 + kRowStep * c < left;
            const int64_t from = c * kRowStep * row_bytes;
            copy_async_or_zero(stage + k_place<D>(row0 + kRowStep * c, chunk0), k + from, real);
            copy_async_or_zero(stage + S::kTileBytes + v_place<D>(row0 + kRowStep * c, chunk0), v + from, real);
          }
        }
        if (lane < 2 && at >= 0)
          copy_async<4>(stage + 2 * S::kTileBytes + 4 * lane,
                        (lane == 0 ? a.scale[0] : a.scale[1]) + (int64_t)scale * a.kv_heads + seg.head);
      }
      copy_commit();
    };

#pragma unroll 1  // code that runs once is fetched cold: the less of it the better
    for (int i = 0; i < S::kEarly; ++i) issue(i, i);
    bool first = true;
    while (true) {
#pragma unroll 1
      for (int i = S::kEarly; i < S::kStages - 1; ++i) issue(i, i);
      // While the first tiles are on their way: the segment after this one, and q.
      walk.advance(a);
      more = walk.next(a, &coming);
      if (more) {
        fetch_queries(coming, walk.seq, both - queries);
        page_coming = page_of(coming, keys_of(coming, walk.seq), 0);
      }
      // The fewest keys that a row sees: tiles below it need no mask.
      const int fewest = max(0, seq.context - seq.q_len + seg.tile * a.rows / a.group + 1);
      const int count = seg.end - seg.begin;
      int stage_now = 0;
      Rows<D, NT> r;
      if (first) {  // else they came with the last segment's tiles
        copy_wait<S::kStages - 1>();
        __syncthreads();
        first = false;
      }
      load_rows<D, NT>(a, seq, seg, queries, g, t, r);

      for (int i = 0; i < count; ++i) {
        issue(i + S::kStages - 1, stage_now == 0 ? S::kStages - 1 : stage_now - 1);
        copy_wait<S::kStages - 1>();
        __syncwarp();
        const int tile = (seg.begin + i) * kWarps + warp;
        const int behind = min(S::kStages - 1, count - 1 - i);  // tiles issued after this one
        if (tile * kTile < keys && (absent >> behind & 1) == 0) {
          const uint32_t stage = ring + stage_now * S::kStageBytes;
          const float2 scales = load_shared_f2(stage + 2 * S::kTileBytes);
          float x[NT][4], odd[NT][4];  // two chains of products, half as long
#pragma unroll
          for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int k = 0; k < 4; ++k) x[j][k] = odd[j][k] = 0.0f;
#pragma unroll
          for (int c = 0; c < D / 64; ++c) {
            const uint4 lo = load_shared16(stage + k_place<D>(g, 4 * c + t));
            const uint4 hi = load_shared16(stage + k_place<D>(g + 8, 4 * c + t));
            const uint32_t low[4] = {lo.x, lo.y, lo.z, lo.w}, high[4] = {hi.x, hi.y, hi.z, hi.w};
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const uint32_t a0 = widen_low(low[k]), a1 = widen_low(high[k]);
              const uint32_t a2 = widen_high(low[k]), a3 = widen_high(high[k]);
#pragma unroll
              for (int j = 0; j < NT; ++j)
                mma(k % 2 == 0 ? x[j] : odd[j], a0, a1, a2, a3, r.q[j][4 * c + k][0], r.q[j][4 * c + k][1]);
            }
          }
          VTile<D> v;
          v.load(stage + S::kTileBytes, g, t);

          // Scores in log2 units; x[j][k] is key g + 8 (k / 2), column 2t + k % 2.
          const bool masked = (tile + 1) * kTile > fewest;
          const float v_log2 = scale_log2_of(scales.y);
          float weight[NT][2];  // scale / 2^t
          bool raise = v_log2 > r.far;
#pragma unroll
          for (int j = 0; j < NT; ++j) {
            float most[2];
#pragma unroll
            for (int k = 0; k < 2; ++k) {  // scores above it raise m or t; not a bit higher for a large m
              most[k] = __fadd_rd(r.m[j][k], fminf(kRaise, r.unit[j][k] + (kWeightLog2 + kRaise) - v_log2));
              weight[j][k] = weight_of(v_log2 - r.unit[j][k]);
            }
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              x[j][k] = (x[j][k] + odd[j][k]) * (scales.x * r.factor[j][k & 1]);
              if (masked && tile * kTile + g + 8 * (k >> 1) >= r.limit[j][k & 1])
                x[j][k] = __uint_as_float(kNegInf);
              raise = raise || x[j][k] > most[k & 1];
            }
          }
          if (__any_sync(0xFFFFFFFFu, raise)) {
            const uint32_t filled = v.filled();
            const bool some_empty = filled != 0xFFFFu;
            float least = 1e30f;  // of the units
            const bool empty[2] = {(filled >> g & 1) == 0, (filled >> (g + 8) & 1) == 0};
#pragma unroll
            for (int j = 0; j < NT; ++j) {
              float keep[2];
#pragma unroll
              for (int k = 0; k < 2; ++k) {
                float most = column_most(fmaxf(x[j][k], x[j][k + 2])), most_filled = most;
                const float m = r.m[j][k], unit = r.unit[j][k];
                most = fmaxf(most, m);
                if (most != m) r.l[j][k] *= exp2_fast(m - most);
                if (some_empty) {
                  // Keys of zeros count in l and are taken out: they add nothing to o,
                  // and P with their scale may not fit f16.
                  const float base = most == __uint_as_float(kNegInf) ? 0.0f : most;
#pragma unroll
                  for (int n = 0; n < 2; ++n)
                    if (empty[n]) {
                      r.l[j][k] += exp2_fast(x[j][k + 2 * n] - base);
                      x[j][k + 2 * n] = __uint_as_float(kNegInf);
                    }
                  most_filled = column_most(fmaxf(x[j][k], x[j][k + 2]));
                }
                // All against m, which may be too large for sums with t.
                // (-inf) - (-inf) and inf - inf, of a row that has seen nothing or infinities, are none.
                const float moved = unit + (m - most), term = (most_filled - most) + v_log2 - kWeightLog2;
                const float next = fmaxf(fmaxf(moved, term), kLeastUnit);
                keep[k] = most == m && next == unit ? 1.0f : exp2_fast(moved - next);
                r.m[j][k] = most;
                r.unit[j][k] = next;
                weight[j][k] = weight_of(v_log2 - next);
                if (most != __uint_as_float(kNegInf)) least = fminf(least, next);
                // The tile's scores are 2^-112 of m or less then: l does not notice.
                const float excess = v_log2 - next - kMostWeight;
                if (excess > 0.0f) x[j][k] += excess, x[j][k + 2] += excess;
              }
#pragma unroll
              for (int n = 0; n < kSteps; ++n)
#pragma unroll
                for (int k = 0; k < 4; ++k) r.o[n][j][k] *= keep[k & 1];
            }
            least = fminf(least, __shfl_xor_sync(0xFFFFFFFFu, least, 1));
            r.far = fminf(least, __shfl_xor_sync(0xFFFFFFFFu, least, 2)) + kMostWeight;
          }
          uint32_t p[NT][2], seen[NT][2];
#pragma unroll
          for (int j = 0; j < NT; ++j) {
            float e[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const float m = r.m[j][k & 1];
              // A column that has seen nothing has m = -inf, and x = -inf too.
              e[k] = exp2_fast(x[j][k] - (m == __uint_as_float(kNegInf) ? 0.0f : m));
              r.l[j][k & 1] += e[k];
            }
            p[j][0] = transpose8x8(pack_half(e[0] * weight[j][0], e[1] * weight[j][1]));
            p[j][1] = transpose8x8(pack_half(e[2] * weight[j][0], e[3] * weight[j][1]));
          }
          // Only a tile that the rows see to different lengths can hold NaN that a
          // row must not meet: behind the context there are zeros.
          bool nan = false;
          if (masked && fewest < keys) {
#pragma unroll
            for (int k = 0; k < 4; ++k)
#pragma unroll
              for (int n = 0; n < VTile<D>::kWords; ++n)
                nan = nan || __vcmpeq4(v.w[k][n] & 0x7F7F7F7Fu, 0x7F7F7F7Fu) != 0;
            nan = __any_sync(0xFFFFFFFFu, nan);
          }
          if (__builtin_expect(nan, 0)) {
#pragma unroll
            for (int j = 0; j < NT; ++j) {
              bool see[4];
#pragma unroll
              for (int k = 0; k < 4; ++k)
                see[k] = tile * kTile + g + 8 * (k >> 1) < r.limit[j][k & 1];
              seen[j][0] = transpose8x8((see[0] ? 0x3C00u : 0) | (see[1] ? 0x3C000000u : 0));
              seen[j][1] = transpose8x8((see[2] ? 0x3C00u : 0) | (see[3] ? 0x3C000000u : 0));
            }
            nan_tile<D, NT>(v, p, seen, r);
          } else {
#pragma unroll
            for (int n = 0; n < kSteps; ++n) {
              uint32_t f[4];
              v.fragment(n, f);
#pragma unroll
              for (int j = 0; j < NT; ++j) mma(r.o[n][j], f[0], f[1], f[2], f[3], p[j][0], p[j][1]);
            }
          }
        }
        stage_now = stage_now == S::kStages - 1 ? 0 : stage_now + 1;
        __syncwarp();  // the stage is read before it is filled again
      }
      copy_wait<0>();
      if (!a.direct) launch_dependents();
      const Sequence done_seq = seq;
      const Segment done = seg;
      if (more) {  // its first tiles are on their way while the warps are joined
        seg = coming;
        seq = walk.seq;
        keys = keys_of(seg, seq);
        look_up(seg, 0, page_coming);
        queries = both - queries;
#pragma unroll 1
        for (int i = 0; i < S::kEarly; ++i) issue(i, i);
      }

      // Join the warps: maxima first, then the sums at the common maximum.
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          float l = r.l[j][k];
          l += __shfl_xor_sync(0xFFFFFFFFu, l, 4);
          l += __shfl_xor_sync(0xFFFFFFFFu, l, 8);
          l += __shfl_xor_sync(0xFFFFFFFFu, l, 16);
          r.l[j][k] = l;
          if (g == 0) {
            warp_m[warp][8 * j + 2 * t + k] = r.m[j][k];
            warp_l[warp][8 * j + 2 * t + k] = l;
          }
        }
      constexpr int kPitch = S::kPitch;
      float* sums = reinterpret_cast<float*>(shared + warp * S::kWarpBytes + S::kSumsAt);
      __syncthreads();
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const int column = 8 * j + 2 * t + k;
          float most = warp_m[0][column];
#pragma unroll
          for (int w = 1; w < kWarps; ++w) most = fmaxf(most, warp_m[w][column]);
          const float m = r.m[j][k];
          const float keep = m == __uint_as_float(kNegInf) ? 0.0f : exp2_fast(m - most + r.unit[j][k]);
#pragma unroll
          for (int n = 0; n < kSteps; ++n)
            *reinterpret_cast<float2*>(sums + column * kPitch + D / 8 * g + 2 * n) =
                make_float2(r.o[n][j][k] * keep, r.o[n][j][k + 2] * keep);
        }
      __syncthreads();
      const int rows = min(a.rows, done_seq.q_len * a.group - done.tile * a.rows);
      float* slot = done.whole ? nullptr
                               : a.partial + ((int64_t)walk.cta * 2 + done.slot) * slot_floats(a.rows, D);
      for (int i = threadIdx.x; i < rows * (D / 2); i += kThreads) {
        const int row = i / (D / 2), d = i % (D / 2) * 2;
        const float* from = reinterpret_cast<const float*>(shared + S::kSumsAt) + row * kPitch + d;
        float most = warp_m[0][row];
#pragma unroll
        for (int w = 1; w < kWarps; ++w) most = fmaxf(most, warp_m[w][row]);
        float2 sum = make_float2(0.0f, 0.0f);
        float l = 0.0f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
          const float2 x = *reinterpret_cast<const float2*>(from + w * (S::kWarpBytes / 4));
          sum.x += x.x;
          sum.y += x.y;
          // A row that has seen nothing but NaN has no maximum, and its sum is NaN.
          l += (most == __uint_as_float(kNegInf) ? 1.0f : exp2_fast(warp_m[w][row] - most)) * warp_l[w][row];
        }
        if (done.whole) {
          const int at = done.tile * a.rows + row;
          const int token = done_seq.start + at / a.group, head = done.head * a.group + at % a.group;
          const float scale = l == 0.0f ? 0.0f : 1.0f / l;
          write_pair(a, token, head, D, d, sum.x * scale, sum.y * scale);
          if (d == 0) write_lse(a, token, head, most, l);
        } else {
          *reinterpret_cast<float2*>(slot + row * D + d) = sum;
          if (d == 0) {
            slot[a.rows * D + row] = most;
            slot[a.rows * D + a.rows + row] = l;
          }
        }
      }
      if (!more) break;
      __syncthreads();  // the sums are read before the next segment fills their stages
    }
  }
  if (threadIdx.x == 0) walk.finish(a);
}

template <int D, int NT>
int launch(const Args& a, int grid, cudaStream_t stream) {
  constexpr int kBytes = Shape<D, NT>::kBytes;
  static_assert(kBytes <= 224 * 1024, "shared memory");
  KVOFF_TRY((allow_shared<attention_decode_fp8_kernel<D, NT>>(kBytes)));
  attention_decode_fp8_kernel<D, NT><<<grid, kThreads, kBytes, stream>>>(a);
  return cuda_status(cudaGetLastError(), "attention_fp8 launch");
}

}  // namespace

int launch_decode(const Args& a, int dim, int grid, cudaStream_t stream) {
  if (dim == 128) return a.rows == 8 ? launch<128, 1>(a, grid, stream) : launch<128, 2>(a, grid, stream);
  return a.rows == 8 ? launch<64, 1>(a, grid, stream) : launch<64, 2>(a, grid, stream);
}

}  // namespace attention
}  // namespace kvoff
