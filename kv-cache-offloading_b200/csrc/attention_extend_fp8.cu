// Attention of many query rows over the e4m3 paged cache (prompt chunks over a
// cached history): 256 packed rows of one KV head against 128 keys at a time
// on the tensor cores, accumulators in tensor memory.
//
// Bound by the matrix products (4 D flops per visible row and key; the cache
// is read once per 256 rows, mostly from L2) and next by the exponentials: 128
// x 128 of them take the special function units as long as the two products
// of the tile take the tensor cores (1024 cycles). So two 128-row tiles run in
// turn: while one's scores go through the softmax, the other's products run,
// and each key tile is converted once for both.
//
//   warps 0-3, 4-7  softmax of row tile 0 and 1, one row a thread
//   warps 8-11      cache -> registers -> f16 operands in shared memory
//   warp 12         one thread issues all matrix products
//
// K, V and Q are f16 operands: e4m3 is a subset of f16, and q is scaled by a
// power of two to an amax of 2^14..2^15, where every bf16 value down to 2^-31
// of the row's largest is exact. The scores S = Q K^T are fp32 in tensor
// memory; a scale block is 16 tokens or more, so the scale of K enters once
// per 16 scores. P = exp2(x - m) takes the scale of V with it, as a fraction
// of the largest met so far (bias in the exponent), times 2^8, and goes back
// to tensor memory as the f16 operand of O += P V, in the place of its scores.
// The sum of p is taken before that, per 16 keys, and divided by the same
// factor. The maximum is raised only when a score passes it by 2^6, so the
// accumulator is rescaled a few times in a row tile, not once in each key tile.
//
// Order: s_full (scores of tile j) implies that all products issued before
// them are complete, O of tile j - 1 among them, so a softmax thread may
// rescale its row of O at any time before it reports P.
//
// Every wait is bounded; one that runs out sets an error flag that
// kvoff_device_error reads, and all roles leave.
#include "attention_fp8.h"
#include "codec.cuh"

namespace kvoff {
namespace attention {

__device__ int g_extend_error = 0;

namespace {

constexpr int kThreads = 512;
constexpr int kGroupRows = 128;    // rows of a tensor tile
constexpr int kStages = 2;         // of K and of V
constexpr int kScaleRing = 4;      // scales live longer than K's stage
constexpr float kRaise = 6.0f;     // log2 of how far P may pass 1
constexpr float kWeightLog2 = 8.0f;
constexpr float kLeastLog2 = -42.0f;  // of a V scale against the largest: P rounds to 0 in f16
constexpr uint32_t kNegInf = 0xFF800000u;
constexpr uint64_t kWaitLimitNs = 1000000000ull;
constexpr uint32_t kTmemColumns = 512;
constexpr uint32_t kScoresAt = 0, kOutputsAt = 256, kGroupColumns = 128;

template <int D>
struct Layout {
  static constexpr int kOperand = 128 * D * 2;  // bytes of a 128-row f16 tile
  static constexpr int kQ = 0;
  static constexpr int kK = kQ + 2 * kOperand;
  static constexpr int kV = kK + kStages * kOperand;
  static constexpr int kNan = kV + kStages * kOperand;  // [stage][key][D / 16] 16-bit masks
  static constexpr int kNanBytes = 128 * (D / 16) * 2;
  static constexpr int kBytes = kNan + kStages * kNanBytes + 1024;  // 1024: alignment
};

struct Scales {
  float k[8];       // of the tile's 16-key groups
  float v_log2[8];
  uint32_t absent;  // bit g: group g has no page
};

struct Shared {
  uint64_t q_full[2], s_full[2], p_full[2], o_full[2];
  uint64_t k_full[kStages], k_empty[kStages], v_full[kStages], v_empty[kStages];
  uint64_t scale_full[kScaleRing];
  uint64_t drained;
  Scales scales[kScaleRing];
  uint32_t nan[kStages];  // n + 1: V of tile n, in this stage, holds NaN that some row must not meet
  uint32_t tmem;
  int32_t abort;
  Walk<kThreads>::Shared walk;
  // Each warp's place in the CTA's work, here rather than in registers: one
  // lane moves it, once a segment.
  struct Place {
    Walk<kThreads> walk;
    Segment segment;
  } place[kThreads / 32];
};

__device__ __forceinline__ uint32_t smem_of(const void* p) {
  return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}

__device__ __forceinline__ void bar_init(uint64_t* bar, uint32_t count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_of(bar)), "r"(count) : "memory");
}
__device__ __forceinline__ void bar_arrive(uint64_t* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_of(bar)) : "memory");
}
__device__ __forceinline__ bool bar_try(uint64_t* bar, uint32_t parity) {
  uint32_t done;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(done)
      : "r"(smem_of(bar)), "r"(parity)
      : "memory");
  return done != 0;
}

// Waits for the phase of `parity`, at most kWaitLimitNs and not once another
// role has given up. False: leave.
__device__ __noinline__ bool bar_wait_slow(uint64_t* bar, uint32_t parity, int32_t* abort) {
  uint64_t begin, now;
  asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(begin));
  for (uint32_t spins = 0; spins < 1u << 26; ++spins) {
    if (bar_try(bar, parity)) return true;
    if (*reinterpret_cast<volatile int32_t*>(abort) != 0) return false;
    asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(now));
    if (now - begin > kWaitLimitNs) break;
  }
  *reinterpret_cast<volatile int32_t*>(abort) = 1;
  atomicOr(&g_extend_error, kErrExtendWaitTimeout);
  return false;
}
__device__ __forceinline__ bool bar_wait(uint64_t* bar, uint32_t parity, int32_t* abort) {
  if (bar_try(bar, parity)) return true;
  return bar_wait_slow(bar, parity, abort);
}
// The same for a whole warp, whose lanes stay or leave together.
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, int32_t* abort) {
  return __all_sync(0xFFFFFFFFu, bar_wait(bar, parity, abort));
}

__device__ __forceinline__ void tensor_fence_before() {
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
}
__device__ __forceinline__ void tensor_fence_after() {
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
}
__device__ __forceinline__ void async_fence() {
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
}
__device__ __forceinline__ void commit(uint64_t* bar) {
  asm volatile(
      "tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_of(bar))
      : "memory");
}

// Operands in shared memory: blocks of 64 f16 columns (128 bytes), 16-byte
// chunk c of row r at chunk c ^ (r % 8), rows 128 bytes apart; blocks follow
// one another 128 rows apart.
constexpr uint64_t kDescriptor = (uint64_t)1 << 46      // version
                                 | (uint64_t)2 << 61    // 128-byte swizzle
                                 | (uint64_t)(1024 >> 4) << 32;  // from 8 rows to the next 8
// K-major (the reduction runs along a row): the leading offset is not used.
__device__ __forceinline__ uint64_t row_descriptor(uint32_t address) {
  return kDescriptor | (uint64_t)1 << 16 | address >> 4;
}
// MN-major (the reduction runs over rows): the leading offset leads from one
// 64-column block to the next.
__device__ __forceinline__ uint64_t column_descriptor(uint32_t address) {
  return kDescriptor | (uint64_t)(16384 >> 4) << 16 | address >> 4;
}

// f16 operands, fp32 sums, M = 128; B is N x K along K, or along N.
template <int N, bool kBColumns>
constexpr uint32_t kInstruction = 1u << 4 | (kBColumns ? 1u << 16 : 0u) | (uint32_t)(N / 8) << 17 |
                                  (uint32_t)(128 / 16) << 24;

__device__ __forceinline__ void mma_shared(uint32_t d, uint64_t a, uint64_t b, uint32_t instruction,
                                           bool add) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(instruction), "r"((uint32_t)add)
      : "memory");
}
__device__ __forceinline__ void mma_tensor(uint32_t d, uint32_t a, uint64_t b, uint32_t instruction,
                                           bool add) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(a), "l"(b), "r"(instruction), "r"((uint32_t)add)
      : "memory");
}

#define KVOFF_LIST4(op, a, i) op(a[(i)]), op(a[(i) + 1]), op(a[(i) + 2]), op(a[(i) + 3])
#define KVOFF_LIST16(op, a, i) \
  KVOFF_LIST4(op, a, i), KVOFF_LIST4(op, a, (i) + 4), KVOFF_LIST4(op, a, (i) + 8), KVOFF_LIST4(op, a, (i) + 12)
#define KVOFF_OUT(x) "=f"(x)
#define KVOFF_THROUGH(x) "+f"(x)
#define KVOFF_IN(x) "r"(x)
#define KVOFF_IN_F(x) "f"(x)

// 32 columns of this thread's row, between begin and end on their way. The wait
// passes them through, so that nothing that uses them can be moved before it.
__device__ __forceinline__ void load_begin(float (&x)[32], uint32_t from) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,"
      "%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : KVOFF_LIST16(KVOFF_OUT, x, 0), KVOFF_LIST16(KVOFF_OUT, x, 16)
      : "r"(from)
      : "memory");
}
__device__ __forceinline__ void load_end(float (&x)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : KVOFF_LIST16(KVOFF_THROUGH, x, 0), KVOFF_LIST16(KVOFF_THROUGH, x, 16)::"memory");
}
__device__ __forceinline__ void tensor_store16(uint32_t to, const uint32_t (&x)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,"
      "%13,%14,%15};" ::KVOFF_LIST16(KVOFF_IN, x, 0),
      "r"(to)
      : "memory");
}
// Eight columns times `by`, in place.
__device__ __forceinline__ void tensor_scale8(uint32_t at, float by) {
  float x[8];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : KVOFF_LIST4(KVOFF_OUT, x, 0), KVOFF_LIST4(KVOFF_OUT, x, 4)
      : "r"(at)
      : "memory");
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] *= by;
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%8], {%0,%1,%2,%3,%4,%5,%6,%7};" ::KVOFF_LIST4(
                   KVOFF_IN_F, x, 0),
               KVOFF_LIST4(KVOFF_IN_F, x, 4), "r"(at)
               : "memory");
}
__device__ __forceinline__ void tensor_wait_stores() {
  asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t pack_half(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ uint32_t widen(uint32_t pair) {  // two e4m3 -> f16x2, exact
  uint32_t r;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"((uint16_t)pair));
  return r;
}

// What of a segment all roles agree on.
struct View {
  int keys;    // that the last row sees: nothing is read behind them
  int fewest;  // that the first row sees
  int rows;
  __device__ __forceinline__ View(const Args& a, const Sequence& seq, const Segment& seg) {
    keys = min(seq.keys(a, seg.tile), seq.context);
    fewest = max(0, seq.context - seq.q_len + seg.tile * a.rows / a.group + 1);
    rows = min(a.rows, seq.q_len * a.group - seg.tile * a.rows);
  }
  __device__ __forceinline__ int groups() const { return rows > kGroupRows ? 2 : 1; }
  // Whether rows see key tile `tile` to different lengths.
  __device__ __forceinline__ bool mixed(int tile) const {
    return (tile + 1) * kKeyTile > fewest && fewest < keys;
  }
};

// Chunk `chunk` (8 f16 values) of row `row` of an operand.
template <int D>
__device__ __forceinline__ uint32_t operand_at(int row, int chunk) {
  return (chunk / 8) * 16384 + row * 128 + ((chunk % 8) ^ (row % 8)) * 16;
}
__device__ __forceinline__ void store_shared(uint32_t to, uint4 v) {
  asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(to), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w)
               : "memory");
}

// The warp's next segment, whose sequence is walk.seq, or false.
__device__ __forceinline__ bool next_segment(const Args& a, Shared::Place& place, bool first) {
  bool more = false;
  __syncwarp();
  if (threadIdx.x % 32 == 0) {
    if (!first) place.walk.advance(a);
    more = place.walk.next(a, &place.segment);
  }
  __syncwarp();
  return __any_sync(0xFFFFFFFFu, more);
}

__device__ __forceinline__ uint4 load_shared(uint32_t p) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "r"(p)
               : "memory");
  return v;
}
__device__ __forceinline__ uint32_t pack_out(const Args& a, float x, float y) {
  uint32_t r;
  if (a.bf16)
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(y), "f"(x));
  else
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(y), "f"(x));
  return r;
}

// --- warps 8-11 ------------------------------------------------------------

template <int D>
struct Convert {
  static constexpr int kChunks = D / 16;         // 16-byte chunks of a row
  static constexpr int kPasses = kChunks;        // 128 threads over 128 rows
  static constexpr int kRowsAPass = 128 / kChunks;
  const Args& a;
  Shared* sh;
  uint32_t base;
  int t;  // thread of the warpgroup

  // The group (16 keys) that pass i of this thread reads.
  __device__ __forceinline__ int row(int i) const { return t / kChunks + kRowsAPass * i; }

  __device__ __forceinline__ void load(int kv, const View& view, const Segment& seg, int tile, int page_of,
                                       uint4 (&raw)[kPasses]) const {
    const int chunk = t % kChunks;
    const uint8_t* cache = kv != 0 ? a.cache[1] : a.cache[0];
    const int64_t row_bytes = (int64_t)a.kv_heads * D;
#pragma unroll
    for (int i = 0; i < kPasses; ++i) {
      const int r = row(i), key = tile * kKeyTile + r;
      const int page = __shfl_sync(0xFFFFFFFFu, page_of, r / 16);
      raw[i] = make_uint4(0, 0, 0, 0);
      if (key < view.keys && page >= 0)
        raw[i] = __ldg(reinterpret_cast<const uint4*>(
            cache + ((int64_t)page * a.page + key % a.page) * row_bytes + seg.head * D + chunk * 16));
    }
  }

  __device__ __forceinline__ void put(uint32_t to, const uint4 (&raw)[kPasses]) const {
    const int chunk = t % kChunks;
#pragma unroll
    for (int i = 0; i < kPasses; ++i) {
      const uint4 lo = make_uint4(widen(raw[i].x & 0xFFFFu), widen(raw[i].x >> 16),
                                  widen(raw[i].y & 0xFFFFu), widen(raw[i].y >> 16));
      const uint4 hi = make_uint4(widen(raw[i].z & 0xFFFFu), widen(raw[i].z >> 16),
                                  widen(raw[i].w & 0xFFFFu), widen(raw[i].w >> 16));
      // The threads of the second block of a row write their halves in the
      // other order: eight threads meet all banks.
      const bool swap = chunk >= 4;
      store_shared(to + operand_at<D>(row(i), 2 * chunk + swap), swap ? hi : lo);
      store_shared(to + operand_at<D>(row(i), 2 * chunk + !swap), swap ? lo : hi);
    }
  }

  // Takes NaN out of V and notes them, one bit each, per key and chunk.
  __device__ __forceinline__ void take_nan(int stage, uint32_t count, uint4 (&raw)[kPasses], uint8_t* masks) const {
    const int chunk = t % kChunks;
#pragma unroll
    for (int i = 0; i < kPasses; ++i) {
      uint32_t w[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
      uint32_t mask = 0;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const uint32_t is = __vcmpeq4(w[k] & 0x7F7F7F7Fu, 0x7F7F7F7Fu);
        w[k] &= ~is;
        mask |= ((is & 1u) | (is >> 7 & 2u) | (is >> 14 & 4u) | (is >> 21 & 8u)) << 4 * k;
      }
      raw[i] = make_uint4(w[0], w[1], w[2], w[3]);
      reinterpret_cast<uint16_t*>(masks)[row(i) * kChunks + chunk] = (uint16_t)mask;
      if (mask != 0) *reinterpret_cast<volatile uint32_t*>(&sh->nan[stage]) = count + 1;
    }
  }
};

template <int D>
__device__ __forceinline__ void convert_role(const Args& a, Shared::Place& place, Shared* sh, uint8_t* smem) {
  Convert<D> c{a, sh, smem_of(smem), (int)threadIdx.x % 128};
  constexpr int kPasses = Convert<D>::kPasses;
  using L = Layout<D>;
  const int lane = threadIdx.x % 32;
  const int blocks = a.page / 16 / a.block_tiles;  // scale blocks of a page
  uint32_t count = 0;  // key tiles so far, over all segments
  for (bool first = true; next_segment(a, place, first); first = false) {
    const Segment seg = place.segment;
    const View view(a, place.walk.seq, seg);
    const int32_t* table = a.tables + seg.seq * a.table_stride;
    // Lane g < 8 of each warp holds the page of group g of a tile, -1 for none.
    auto page_of = [&](int tile) {
      const int key = tile * kKeyTile + lane * 16;
      int id = -1;
      if (lane < 8 && tile < seg.end && key < view.keys) {
        id = __ldg(table + key / a.page);
        if (id >= a.num_pages) id = -1;
      }
      return id < 0 ? -1 : id;
    };
    float k_scale = 0.0f, v_scale = 0.0f;
    uint32_t absent = 0;
    auto load_scales = [&](int tile, int page) {
      k_scale = v_scale = 0.0f;
      const int key = tile * kKeyTile + lane * 16;
      if (page >= 0) {
        const int64_t at =
            ((int64_t)page * blocks + key % a.page / 16 / a.block_tiles) * a.kv_heads + seg.head;
        k_scale = __ldg(a.scale[0] + at);
        v_scale = __ldg(a.scale[1] + at);
      }
      absent = __ballot_sync(0xFFFFFFFFu, page < 0) & 0xFFu;
    };
    uint4 k_raw[kPasses], v_raw[kPasses];
    int page = page_of(seg.begin), page_next = page_of(seg.begin + 1);
    c.load(0, view, seg, seg.begin, page, k_raw);
    c.load(1, view, seg, seg.begin, page, v_raw);
    load_scales(seg.begin, page);
    for (int tile = seg.begin; tile < seg.end; ++tile, ++count) {
      const int stage = count % kStages;
      const uint32_t parity = (count / kStages & 1) ^ 1;
      if (!warp_wait(&sh->k_empty[stage], parity, &sh->abort)) return;
      c.put(c.base + L::kK + stage * L::kOperand, k_raw);
      if (c.t < 32) {
        Scales& s = sh->scales[count % kScaleRing];
        if (lane < 8) {
          s.k[lane] = k_scale;
          s.v_log2[lane] = v_scale > 0.0f ? log2f(v_scale) : v_scale == v_scale ? -200.0f : v_scale;
        }
        if (lane == 0) s.absent = absent;
        __syncwarp();
        if (lane == 0) bar_arrive(&sh->scale_full[count % kScaleRing]);
      }
      async_fence();
      bar_arrive(&sh->k_full[stage]);
      const bool more = tile + 1 < seg.end;
      page = page_next;
      if (more) {
        page_next = page_of(tile + 2);
        c.load(0, view, seg, tile + 1, page, k_raw);
        load_scales(tile + 1, page);
      }
      if (!warp_wait(&sh->v_empty[stage], parity, &sh->abort)) return;
      if (view.mixed(tile)) {
        c.take_nan(stage, count, v_raw, smem + L::kNan + stage * L::kNanBytes);
      }
      c.put(c.base + L::kV + stage * L::kOperand, v_raw);
      async_fence();
      bar_arrive(&sh->v_full[stage]);
      if (more) c.load(1, view, seg, tile + 1, page, v_raw);
    }
  }
}

// --- warp 12 ---------------------------------------------------------------

template <int D>
__device__ __forceinline__ void issue_role(const Args& a, Shared::Place& place, Shared* sh, uint32_t base) {
  using L = Layout<D>;
  const uint32_t tmem = sh->tmem;
  uint32_t count = 0, turn[2] = {0, 0}, segment[2] = {0, 0};
  auto scores = [&](int g, int stage) {
#pragma unroll
    for (int k = 0; k < D / 16; ++k) {
      const uint32_t at = (k / 4) * 16384 + (k % 4) * 32;
      mma_shared(tmem + kScoresAt + g * kGroupColumns, row_descriptor(base + L::kQ + g * L::kOperand + at),
                 row_descriptor(base + L::kK + stage * L::kOperand + at), kInstruction<128, false>, k > 0);
    }
    commit(&sh->s_full[g]);
  };
  for (; place.walk.next(a, &place.segment); place.walk.advance(a)) {
    const Segment seg = place.segment;
    const View view(a, place.walk.seq, seg);
    const int groups = view.groups(), tiles = seg.end - seg.begin;
    if (!bar_wait(&sh->k_full[count % kStages], count / kStages & 1, &sh->abort)) return;
    for (int g = 0; g < groups; ++g) {
      if (!bar_wait(&sh->q_full[g], segment[g] & 1, &sh->abort)) return;
      ++segment[g];
      tensor_fence_after();
      scores(g, count % kStages);
    }
    commit(&sh->k_empty[count % kStages]);
    for (int i = 0; i < tiles; ++i, ++count) {
      const int stage = count % kStages, next = (count + 1) % kStages;
      if (!bar_wait(&sh->v_full[stage], count / kStages & 1, &sh->abort)) return;
      for (int g = 0; g < groups; ++g) {
        if (!bar_wait(&sh->p_full[g], turn[g] & 1, &sh->abort)) return;
        ++turn[g];
        tensor_fence_after();
#pragma unroll
        for (int k = 0; k < 8; ++k)
          mma_tensor(tmem + kOutputsAt + g * kGroupColumns, tmem + kScoresAt + g * kGroupColumns + k * 8,
                     column_descriptor(base + L::kV + stage * L::kOperand + k * 2048), kInstruction<D, true>,
                     i > 0 || k > 0);
        if (g == groups - 1) commit(&sh->v_empty[stage]);
        if (i + 1 < tiles) {
          if (g == 0 && !bar_wait(&sh->k_full[next], (count + 1) / kStages & 1, &sh->abort)) return;
          tensor_fence_after();
          scores(g, next);
          if (g == groups - 1) commit(&sh->k_empty[next]);
        } else {
          commit(&sh->o_full[g]);
        }
      }
    }
  }
}

// --- warps 0-7 -------------------------------------------------------------

template <int D>
__device__ __forceinline__ void softmax_role(const Args& a, Shared::Place& place, Shared* sh, uint8_t* smem) {
  using L = Layout<D>;
  const int g = threadIdx.x / 128, r = threadIdx.x % 128;
  const uint32_t base = smem_of(smem);
  const uint32_t lanes = (uint32_t)(r / 32 * 32) << 16;
  const uint32_t scores_at = sh->tmem + lanes + kScoresAt + g * kGroupColumns;
  const uint32_t output_at = sh->tmem + lanes + kOutputsAt + g * kGroupColumns;
  uint32_t count = 0, turn = 0, segment = 0;
  for (bool first = true; next_segment(a, place, first); first = false) {
    const Sequence& seq = place.walk.seq;
    const Segment& seg = place.segment;
    const View view(a, seq, seg);
    if (g >= view.groups()) {
      count += seg.end - seg.begin;
      continue;
    }
    const int at = seg.tile * a.rows + g * kGroupRows + r;  // this thread's packed row
    const bool real = g * kGroupRows + r < view.rows;
    const int token = seq.start + at / a.group, head = seg.head * a.group + at % a.group;
    const int limit = real ? max(0, seq.context - seq.q_len + at / a.group + 1) : 0;
    float factor;
    {  // q: one row a thread, scaled to an amax of 2^14..2^15
      const uint4* from =
          reinterpret_cast<const uint4*>(a.q + token * a.q_stride + (int64_t)head * D * 2);
      uint32_t most = 0;
      auto values = [&](const uint4& v, float (&x)[8]) {
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float2 f;
          if (a.bf16)
            f = make_float2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xFFFF0000u));
          else
            f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
          x[2 * i] = f.x, x[2 * i + 1] = f.y;
        }
      };
      uint4 raw[D / 8];
#pragma unroll
      for (int c = 0; c < D / 8; ++c) raw[c] = real ? __ldg(from + c) : make_uint4(0, 0, 0, 0);
#pragma unroll
      for (int c = 0; c < D / 8; ++c) {
        float x[8];
        values(raw[c], x);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const uint32_t u = __float_as_uint(x[i]) & 0x7FFFFFFFu;
          if (u < 0x7F800000u) most = max(most, u);
        }
      }
      const int e = most == 0 ? 0 : min(14 - ((int)(most >> 23) - 127), 100);
      const float up = __uint_as_float((uint32_t)(127 + e) << 23);
      factor = a.scale_log2 * __uint_as_float((uint32_t)(127 - e) << 23);
      const uint32_t to = base + L::kQ + g * L::kOperand;
#pragma unroll
      for (int c = 0; c < D / 8; ++c) {
        float x[8];
        values(raw[c], x);
        store_shared(to + operand_at<D>(r, c),
                     make_uint4(pack_half(x[0] * up, x[1] * up), pack_half(x[2] * up, x[3] * up),
                                pack_half(x[4] * up, x[5] * up), pack_half(x[6] * up, x[7] * up)));
      }
      async_fence();
      tensor_fence_before();
      bar_arrive(&sh->q_full[g]);
    }
    float m = __uint_as_float(kNegInf), l = 0.0f, ref = -200.0f;  // ref: log2 of the largest V scale
    uint32_t nan[D / 32];
#pragma unroll
    for (int i = 0; i < D / 32; ++i) nan[i] = 0;

    for (int tile = seg.begin; tile < seg.end; ++tile, ++count) {
      if (!warp_wait(&sh->s_full[g], turn & 1, &sh->abort)) return;
      ++turn;
      tensor_fence_after();
      const Scales& scales = sh->scales[count % kScaleRing];
      if (!warp_wait(&sh->scale_full[count % kScaleRing], count / kScaleRing & 1, &sh->abort)) return;
      const uint32_t absent = scales.absent;
      const int seen = limit - tile * kKeyTile;  // of this tile's keys
      const bool masked = __any_sync(0xFFFFFFFFu, seen < kKeyTile) || absent != 0;
      auto mask = [&](int c, float (&s)[32]) {
#pragma unroll
        for (int i = 0; i < 32; ++i)
          if (32 * c + i >= seen || (absent >> (2 * c + i / 16) & 1)) s[i] = __uint_as_float(kNegInf);
      };
      // A scale of zero must not meet a masked score's infinity.
      auto factor_of = [&](int b) { return fmaxf(scales.k[b] * factor, 1e-37f); };

      // The row's maximum; then its scores again, which costs less than the
      // registers to keep them.
      float buffer[2][32];
      float most = __uint_as_float(kNegInf), ref_now = ref;
      load_begin(buffer[0], scores_at);
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        float(&s)[32] = buffer[c % 2];
        load_end(s);
        load_begin(buffer[(c + 1) % 2], scores_at + (c + 1) % 4 * 32);
        if (masked) mask(c, s);
#pragma unroll
        for (int b = 0; b < 2; ++b) {
          float top = s[16 * b];
#pragma unroll
          for (int i = 1; i < 16; ++i) top = fmaxf(top, s[16 * b + i]);
          most = fmaxf(most, top * factor_of(2 * c + b));
          ref_now = fmaxf(ref_now, scales.v_log2[2 * c + b]);
        }
      }
      load_end(buffer[0]);
      if (__any_sync(0xFFFFFFFFu, most > m + kRaise || ref_now > ref)) {
        const float top = fmaxf(m, most);
        const float keep_l = top == m ? 1.0f : exp2_fast(m - top);
        if (tile != seg.begin) {
          const float keep = keep_l * exp2_fast(ref - ref_now);
#pragma unroll 1
          for (int c = 0; c < D / 8; ++c) tensor_scale8(output_at + 8 * c, keep);
        }
        l *= keep_l;
        m = top;
        ref = ref_now;
      }
      const float shift = m == __uint_as_float(kNegInf) ? 0.0f : m;
      float scale_log2 = 0.0f, last = 1e30f, unscale = 1.0f;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        float(&s)[32] = buffer[c % 2];
        if (c > 0) load_end(s);
        if (c < 3) load_begin(buffer[(c + 1) % 2], scores_at + (c + 1) * 32);
        if (masked) mask(c, s);
        uint32_t p[16];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const int b = 2 * c + k;
          const float v_log2 = scales.v_log2[b];
          if (v_log2 != last) {  // one number for all of a larger scale block
            last = v_log2;
            const float relative = v_log2 - ref;
            scale_log2 = (relative < kLeastLog2 ? kLeastLog2 : relative) + kWeightLog2;
            unscale = exp2_fast(-scale_log2);
          }
          const float f = factor_of(b), bias = scale_log2 - shift;
          float sum0 = 0.0f, sum1 = 0.0f;
#pragma unroll
          for (int i = 0; i < 16; i += 2) {
            const float x = exp2_fast(fmaf(s[16 * k + i], f, bias));
            const float y = exp2_fast(fmaf(s[16 * k + i + 1], f, bias));
            sum0 += x;
            sum1 += y;
            p[8 * k + i / 2] = pack_half(x, y);
          }
          l = fmaf(sum0 + sum1, unscale, l);
        }
        // P takes the columns of scores that have been read: 16 for these 32.
        tensor_store16(scores_at + 16 * c, p);
      }
      if (view.mixed(tile)) {
        const int stage = count % kStages;
        if (!warp_wait(&sh->v_full[stage], count / kStages & 1, &sh->abort)) return;
        if (*reinterpret_cast<volatile uint32_t*>(&sh->nan[stage]) == count + 1) {
          const uint32_t* masks = reinterpret_cast<const uint32_t*>(smem + L::kNan + stage * L::kNanBytes);
          for (int i = 0; i < min(seen, kKeyTile); ++i)
#pragma unroll
            for (int w = 0; w < D / 32; ++w) nan[w] |= masks[i * (D / 32) + w];
          __syncwarp();
        }
      }
      tensor_wait_stores();
      tensor_fence_before();
      bar_arrive(&sh->p_full[g]);
    }

    if (!warp_wait(&sh->o_full[g], segment & 1, &sh->abort)) return;
    ++segment;
    tensor_fence_after();
    // exp2(ref) may be as small as a scale can be; a row of zero scales is zero.
    const float scale = exp2_fast(ref - kWeightLog2) * (seg.whole ? (l == 0.0f ? 0.0f : 1.0f / l) : 1.0f);
    float* slot = seg.whole ? nullptr : a.partial + ((int64_t)place.walk.cta * 2 + seg.slot) * slot_floats(a.rows, D);
    const int row = g * kGroupRows + r;
    const uint32_t stage_at = base + L::kQ + g * L::kOperand;  // q is not read any more
#pragma unroll
    for (int c = 0; c < D / 32; ++c) {
      float o[32];
      __syncwarp();
      load_begin(o, output_at + 32 * c);
      load_end(o);
#pragma unroll
      for (int i = 0; i < 32; ++i) o[i] = (nan[c] >> i & 1) != 0 ? __uint_as_float(0x7FC00000u) : o[i] * scale;
      if (seg.whole && a.wide_out) {
#pragma unroll
        for (int k = 0; k < 4; ++k)
          store_shared(stage_at + operand_at<D>(r, 4 * c + k),
                       make_uint4(pack_out(a, o[8 * k], o[8 * k + 1]), pack_out(a, o[8 * k + 2], o[8 * k + 3]),
                                  pack_out(a, o[8 * k + 4], o[8 * k + 5]), pack_out(a, o[8 * k + 6], o[8 * k + 7])));
      } else if (seg.whole) {
        if (real)
#pragma unroll
          for (int i = 0; i < 32; i += 2) write_pair(a, token, head, D, 32 * c + i, o[i], o[i + 1]);
      } else if (real) {
        float4* to = reinterpret_cast<float4*>(slot + (int64_t)row * D + 32 * c);
#pragma unroll
        for (int i = 0; i < 8; ++i)
          to[i] = make_float4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
      }
    }
    __syncwarp();
    if (seg.whole && a.wide_out) {  // the warp's 32 rows, D / 8 threads to a row
      const int first_row = g * kGroupRows + r / 32 * 32;
#pragma unroll 4
      for (int i = threadIdx.x % 32; i < 32 * (D / 8); i += 32) {
        const int k = i / (D / 8), chunk = i % (D / 8);
        if (first_row + k < view.rows) {
          const int to = seg.tile * a.rows + first_row + k;
          uint8_t* out = a.out + (seq.start + to / a.group) * a.out_stride +
                         (int64_t)(seg.head * a.group + to % a.group) * D * 2 + chunk * 16;
          *reinterpret_cast<uint4*>(out) = load_shared(stage_at + operand_at<D>(r / 32 * 32 + k, chunk));
        }
      }
    }
    if (real && seg.whole) write_lse(a, token, head, m, l);
    if (real && !seg.whole) {
      slot[(int64_t)a.rows * D + row] = m;
      slot[(int64_t)a.rows * D + a.rows + row] = l;
    }
    __syncwarp();
  }
}

template <int D>
__global__ void __launch_bounds__(kThreads, 1) attention_extend_fp8_kernel(const __grid_constant__ Args a) {
  extern __shared__ uint8_t raw_shared[];
  __shared__ Shared sh;
  uint8_t* smem = raw_shared + (1024 - smem_of(raw_shared) % 1024) % 1024;
  const int warp = threadIdx.x / 32;
  if (threadIdx.x == 0) {
    for (int g = 0; g < 2; ++g) {
      bar_init(&sh.q_full[g], 128);
      bar_init(&sh.s_full[g], 1);
      bar_init(&sh.p_full[g], 128);
      bar_init(&sh.o_full[g], 1);
    }
    for (int i = 0; i < kStages; ++i) {
      bar_init(&sh.k_full[i], 128);
      bar_init(&sh.k_empty[i], 1);
      bar_init(&sh.v_full[i], 128);
      bar_init(&sh.v_empty[i], 1);
    }
    for (int i = 0; i < kScaleRing; ++i) bar_init(&sh.scale_full[i], 1);
    bar_init(&sh.drained, 1);
    sh.abort = 0;
    sh.nan[0] = sh.nan[1] = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 12) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_of(&sh.tmem)),
                 "r"(kTmemColumns)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  {
    const Walk<kThreads> walk(a, &sh.walk);
    if (threadIdx.x % 32 == 0) sh.place[warp].walk = walk;
  }
  tensor_fence_before();
  __syncthreads();
  tensor_fence_after();

  if (warp < 8) {
    softmax_role<D>(a, sh.place[warp], &sh, smem);
    if (threadIdx.x == 0) sh.place[0].walk.finish(a);
  } else if (warp < 12) {
    convert_role<D>(a, sh.place[warp], &sh, smem);
  } else {
    if (threadIdx.x == 12 * 32) {
      issue_role<D>(a, sh.place[warp], &sh, smem_of(smem));
      // Nothing of this CTA's is in flight when its tensor memory is freed.
      commit(&sh.drained);
      bool done = bar_try(&sh.drained, 0);
      for (int spins = 0; !done && spins < 1 << 20; ++spins) done = bar_try(&sh.drained, 0);
      if (!done) atomicOr(&g_extend_error, kErrExtendWaitTimeout);
    }
    __syncwarp();
  }
  tensor_fence_before();
  __syncthreads();
  tensor_fence_after();
  if (warp == 12)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(sh.tmem), "r"(kTmemColumns));
}

template <int D>
int launch(const Args& a, int grid, cudaStream_t stream) {
  const auto kernel = attention_extend_fp8_kernel<D>;
  KVOFF_TRY(cuda_status(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                             Layout<D>::kBytes),
                        "attention_fp8 shared memory"));
  kernel<<<grid, kThreads, Layout<D>::kBytes, stream>>>(a);
  return cuda_status(cudaGetLastError(), "attention_fp8 launch");
}

}  // namespace

int launch_extend(const Args& a, int dim, int grid, cudaStream_t stream) {
  return dim == 128 ? launch<128>(a, grid, stream) : launch<64>(a, grid, stream);
}

int extend_device_error(int32_t* flags, bool clear) {
  int value = 0;
  KVOFF_TRY(cuda_status(cudaMemcpyFromSymbol(&value, g_extend_error, sizeof(value)),
                        "cudaMemcpyFromSymbol (attention error flags)"));
  if (clear && value != 0) {
    const int zero = 0;
    KVOFF_TRY(cuda_status(cudaMemcpyToSymbol(g_extend_error, &zero, sizeof(zero)),
                          "cudaMemcpyToSymbol (attention error flags)"));
  }
  *flags |= value;
  return KVOFF_OK;
}

}  // namespace attention
}  // namespace kvoff
