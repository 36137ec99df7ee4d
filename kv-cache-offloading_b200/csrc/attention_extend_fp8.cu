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
//   warp 13         one thread walks the CTA's part of the work
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
constexpr int kWorkRing = 2;       // segments handed out ahead
constexpr float kRaise = 6.0f;     // log2 of how far P may pass 1
constexpr float kWeightLog2 = 8.0f;
constexpr float kLeastLog2 = -42.0f;  // of a V scale against the largest: P rounds to 0 in f16
constexpr uint32_t kNegInf = 0xFF800000u;
constexpr uint32_t kWaitNs = 1000, kMostWaits = 1u << 20;  // a second in all
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

// Of a tile's 16-key groups. The scale of V is a fraction of the largest one
// that the segment has met, times 2^8: it is added to the exponent of P, and
// its inverse takes it out of the sum of p again.
struct Scales {
  float k[8];
  float shift[8];    // log2
  float inverse[8];
  float largest;     // log2 of the largest scale of V so far
  uint32_t absent;   // bit g: group g has no page
};

// One segment, as the roles need it.
struct Work {
  int32_t begin, end;  // key tiles; end < 0: no more work
  int32_t seq, head;
  int32_t slot;        // of the partial result, -1 when the segment is whole
  int32_t start;       // of the sequence's tokens
  int32_t offset;      // context - q_len: token t sees offset + t + 1 keys
  int32_t first_row, rows;
  int32_t keys;        // that the last row sees: nothing is read behind them
  int32_t fewest;      // that the first row sees
  int32_t pad;

  __device__ __forceinline__ int groups() const { return rows > 128 ? 2 : 1; }
  // Whether rows see key tile `tile` to different lengths.
  __device__ __forceinline__ bool mixed(int tile) const {
    return (tile + 1) * kKeyTile > fewest && fewest < keys;
  }
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
  uint64_t work_full[kWorkRing], work_empty[kWorkRing];
  Work work[kWorkRing];
  Walk<kThreads>::Shared walk;
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
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(done)
      : "r"(smem_of(bar)), "r"(parity), "r"(kWaitNs)
      : "memory");
  return done != 0;
}

// Waits for the phase of `parity`, at most kMostWaits times kWaitNs and not
// once another role has given up. False: leave.
__device__ __forceinline__ bool bar_wait(uint64_t* bar, uint32_t parity, int32_t* abort) {
  for (uint32_t i = 0; !bar_try(bar, parity); ++i) {
    if (*reinterpret_cast<volatile int32_t*>(abort) != 0) return false;
    if (i >= kMostWaits) {
      *reinterpret_cast<volatile int32_t*>(abort) = 1;
      atomicOr(&g_extend_error, kErrExtendWaitTimeout);
      return false;
    }
  }
  return true;
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
__device__ __forceinline__ void tensor_store32(uint32_t to, const float (&x)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,"
      "%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31};" ::
          KVOFF_LIST16(KVOFF_IN_F, x, 0),
      KVOFF_LIST16(KVOFF_IN_F, x, 16), "r"(to)
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

template <int kRegisters>
__device__ __forceinline__ void more_registers() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegisters));
}
template <int kRegisters>
__device__ __forceinline__ void fewer_registers() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegisters));
}
// 512 threads are launched with 128 registers each; the shares of the four
// warpgroups add up to 4 * 128.
constexpr int kSoftmaxRegisters = 152, kConvertRegisters = 112, kIssueRegisters = 96;
static_assert(2 * kSoftmaxRegisters + kConvertRegisters + kIssueRegisters == 4 * 128, "registers");

// Chunk `chunk` (8 f16 values) of row `row` of an operand.
template <int D>
__device__ __forceinline__ uint32_t operand_at(int row, int chunk) {
  return (chunk / 8) * 16384 + row * 128 + ((chunk % 8) ^ (row % 8)) * 16;
}
__device__ __forceinline__ void store_shared(uint32_t to, uint4 v) {
  asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(to), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w)
               : "memory");
}

__device__ __forceinline__ uint4 load_shared(uint32_t p) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "r"(p)
               : "memory");
  return v;
}
// Two values of q, and of out, in a word.
__device__ __forceinline__ float2 unpack(bool bf16, uint32_t w) {
  if (bf16) return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
  return __half22float2(*reinterpret_cast<const __half2*>(&w));
}
__device__ __forceinline__ uint32_t pack_out(const Args& a, float x, float y) {
  uint32_t r;
  if (a.bf16)
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(y), "f"(x));
  else
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(y), "f"(x));
  return r;
}

// The next segment for a warp (or, in the issuing role, a thread), or null.
__device__ __forceinline__ const Work* take_work(Shared* sh, uint32_t n) {
  const Work* work = &sh->work[n % kWorkRing];
  if (!bar_wait(&sh->work_full[n % kWorkRing], n / kWorkRing & 1, &sh->abort) || work->end < 0) return nullptr;
  return work;
}
__device__ __forceinline__ void return_work(Shared* sh, uint32_t n) { bar_arrive(&sh->work_empty[n % kWorkRing]); }

// --- warp 13 ---------------------------------------------------------------

__device__ __forceinline__ void schedule_role(const Args& a, Walk<kThreads>& walk, Shared* sh) {
  uint32_t n = 0;
  Segment seg;
  for (bool more = true; more; ++n) {
    more = walk.next(a, &seg);
    if (!bar_wait(&sh->work_empty[n % kWorkRing], (n / kWorkRing & 1) ^ 1, &sh->abort)) return;
    Work& w = sh->work[n % kWorkRing];
    w.end = -1;
    if (more) {
      const Sequence& seq = walk.seq;
      w.begin = seg.begin, w.end = seg.end;
      w.seq = seg.seq, w.head = seg.head;
      w.slot = seg.whole ? -1 : seg.slot;
      w.start = seq.start, w.offset = seq.context - seq.q_len;
      w.first_row = seg.tile * a.rows;
      w.rows = min(a.rows, seq.q_len * a.group - w.first_row);
      w.keys = min(seq.keys(a, seg.tile), seq.context);
      w.fewest = max(0, w.offset + w.first_row / a.group + 1);
      walk.advance(a);
    }
    bar_arrive(&sh->work_full[n % kWorkRing]);
  }
  walk.finish(a);
}

// --- warps 8-11 ------------------------------------------------------------

// Volatile: it stays where it stands, a key tile ahead of its use.
__device__ __forceinline__ uint4 load_global(const uint8_t* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p));
  return v;
}

template <int D>
struct Convert {
  static constexpr int kChunks = D / 16;  // 16-byte chunks of a row
  static constexpr int kPasses = kChunks;  // 128 threads over 128 rows
  static constexpr int kRowsAPass = 128 / kChunks;
  const Args& a;
  Shared* sh;
  uint32_t base;
  int t;  // thread of the warpgroup

  // Chunk and first row of this thread. Eight threads have four chunks of an
  // even row and of the next one, whose swizzled places in shared memory are
  // all different.
  __device__ __forceinline__ int chunk() const { return D == 128 ? t % 4 + t / 8 % 2 * 4 : t % 4; }
  __device__ __forceinline__ int row0() const { return D == 128 ? t / 32 * 4 + t / 16 % 2 * 2 + t / 4 % 2 : t / 4; }
  __device__ __forceinline__ int row(int i) const { return row0() + kRowsAPass * i; }

  // `place`: in lane g < 8, where 16-key group g begins in the cache (bytes, at
  // this head), or negative when it has no page. `left`: keys of the tile that
  // are read.
  __device__ __forceinline__ void load(int kv, int64_t place, int left, uint4 (&raw)[kPasses]) const {
    const int64_t row_bytes = (int64_t)a.kv_heads * D;
    const uint8_t* from =
        (kv != 0 ? a.cache[1] : a.cache[0]) + row0() % 16 * row_bytes + chunk() * 16;
#pragma unroll
    for (int i = 0; i < kPasses; ++i) {
      const int64_t at = __shfl_sync(0xFFFFFFFFu, place, row(i) / 16);
      raw[i] = make_uint4(0, 0, 0, 0);
      if (row(i) < left && at >= 0) raw[i] = load_global(from + at);
    }
  }

  __device__ __forceinline__ void put(uint32_t to, const uint4 (&raw)[kPasses]) const {
    // The swizzle is the same in all passes: they are 16 or 32 rows apart.
    const uint32_t first = to + operand_at<D>(row0(), 2 * chunk()), second = to + operand_at<D>(row0(), 2 * chunk() + 1);
#pragma unroll
    for (int i = 0; i < kPasses; ++i) {
      store_shared(first + i * kRowsAPass * 128,
                   make_uint4(widen(raw[i].x & 0xFFFFu), widen(raw[i].x >> 16),
                              widen(raw[i].y & 0xFFFFu), widen(raw[i].y >> 16)));
      store_shared(second + i * kRowsAPass * 128,
                   make_uint4(widen(raw[i].z & 0xFFFFu), widen(raw[i].z >> 16),
                              widen(raw[i].w & 0xFFFFu), widen(raw[i].w >> 16)));
    }
  }

  // Takes NaN out of V and notes them, one bit each, per key and chunk.
  __device__ __forceinline__ void take_nan(int stage, uint32_t count, uint4 (&raw)[kPasses], uint8_t* masks) const {
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
      reinterpret_cast<uint16_t*>(masks)[row(i) * kChunks + chunk()] = (uint16_t)mask;
      if (mask != 0) *reinterpret_cast<volatile uint32_t*>(&sh->nan[stage]) = count + 1;
    }
  }
};

template <int D>
__device__ __forceinline__ void convert_role(const Args& a, Shared* sh, uint8_t* smem) {
  Convert<D> c{a, sh, smem_of(smem), (int)threadIdx.x % 128};
  constexpr int kPasses = Convert<D>::kPasses;
  using L = Layout<D>;
  const int lane = threadIdx.x % 32;
  const int blocks = a.page / 16 / a.block_tiles;  // scale blocks of a page
  uint32_t count = 0;  // key tiles so far, over all segments
  for (uint32_t n = 0;; ++n) {
    const Work* work = take_work(sh, n);
    if (__any_sync(0xFFFFFFFFu, work == nullptr)) return;
    const int32_t* table = a.tables + work->seq * a.table_stride;
    const int begin = work->begin, end = work->end, keys = work->keys, head = work->head;
    // Lane g < 8 of each warp has the page of group g of a tile (checked when it
    // is used, a tile later), and from it where the group's rows and scales begin.
    auto page_of = [&](int tile) {
      const int key = tile * kKeyTile + lane * 16;
      return lane < 8 && tile < end && key < keys ? __ldg(table + key / a.page) : -1;
    };
    int page_next = page_of(begin);
    int64_t place = -1;
    float k_scale = 0.0f, v_scale = 0.0f, largest = -200.0f;
    uint32_t absent = 0;
    uint4 k_raw[kPasses], v_raw[kPasses];
    // Tile `tile` is put into shared memory while tile + 1 is loaded.
#pragma unroll 1
    for (int tile = begin - 1; tile < end; ++tile) {
      if (tile >= begin) {
        const int stage = count % kStages;
        const uint32_t parity = (count / kStages & 1) ^ 1;
        if (!warp_wait(&sh->k_empty[stage], parity, &sh->abort)) return;
        c.put(c.base + L::kK + stage * L::kOperand, k_raw);
        if (c.t < 32) {
          Scales& s = sh->scales[count % kScaleRing];
          const float log2 = v_scale > 0.0f ? log2f(v_scale) : v_scale == v_scale ? -200.0f : v_scale;
          float most = lane < 8 ? log2 : -200.0f;
#pragma unroll
          for (int d = 4; d > 0; d /= 2) most = fmaxf(most, __shfl_xor_sync(0xFFFFFFFFu, most, d));
          largest = fmaxf(largest, __shfl_sync(0xFFFFFFFFu, most, 0));
          if (lane < 8) {
            const float relative = log2 - largest;
            const float shift = (relative < kLeastLog2 ? kLeastLog2 : relative) + kWeightLog2;
            s.k[lane] = k_scale;
            s.shift[lane] = shift;
            s.inverse[lane] = exp2_fast(-shift);
          }
          if (lane == 0) {
            s.largest = largest;
            s.absent = absent;
          }
          __syncwarp();
          if (lane == 0) bar_arrive(&sh->scale_full[count % kScaleRing]);
        }
        async_fence();
        bar_arrive(&sh->k_full[stage]);
        if (!warp_wait(&sh->v_empty[stage], parity, &sh->abort)) return;
        if (work->mixed(tile)) c.take_nan(stage, count, v_raw, smem + L::kNan + stage * L::kNanBytes);
        c.put(c.base + L::kV + stage * L::kOperand, v_raw);
        async_fence();
        bar_arrive(&sh->v_full[stage]);
        ++count;
      }
      if (tile + 1 < end) {
        const int page = page_next < a.num_pages ? page_next : -1;
        page_next = page_of(tile + 2);
        place = -1;
        k_scale = v_scale = 0.0f;
        if (page >= 0) {
          const int in_page = ((tile + 1) * kKeyTile + lane * 16) % a.page;
          place = ((int64_t)page * a.page + in_page) * a.kv_heads * D + head * D;
          const int64_t at = ((int64_t)page * blocks + in_page / 16 / a.block_tiles) * a.kv_heads + head;
          k_scale = __ldg(a.scale[0] + at);
          v_scale = __ldg(a.scale[1] + at);
        }
        absent = __ballot_sync(0xFFFFFFFFu, page < 0) & 0xFFu;
        c.load(0, place, keys - (tile + 1) * kKeyTile, k_raw);
        c.load(1, place, keys - (tile + 1) * kKeyTile, v_raw);
      }
    }
    __syncwarp();
    if (lane == 0) return_work(sh, n);
  }
}

// --- warp 12 ---------------------------------------------------------------

template <int D>
__device__ __forceinline__ void issue_role(Shared* sh, uint32_t base) {
  using L = Layout<D>;
  const uint32_t tmem = sh->tmem;
  uint32_t count = 0;                // key tiles so far
  uint32_t turn[2] = {0, 0}, segment[2] = {0, 0};
  for (uint32_t n = 0;; ++n) {
    const Work* work = take_work(sh, n);
    if (work == nullptr) return;
    const int groups = work->groups(), tiles = work->end - work->begin;
    return_work(sh, n);
    // Step i: the output of key tile i - 1, then the scores of tile i.
#pragma unroll 1
    for (int i = 0; i <= tiles; ++i) {
      const uint32_t now = count + i, before = now - 1;
#pragma unroll 1
      for (int g = 0; g < groups; ++g) {
        const uint32_t scores = tmem + kScoresAt + g * kGroupColumns, output = tmem + kOutputsAt + g * kGroupColumns;
        if (i > 0) {
          if (!bar_wait(&sh->v_full[before % kStages], before / kStages & 1, &sh->abort)) return;
          uint32_t& t = g == 0 ? turn[0] : turn[1];
          if (!bar_wait(&sh->p_full[g], t & 1, &sh->abort)) return;
          ++t;
          tensor_fence_after();
          const uint64_t v = column_descriptor(base + L::kV + before % kStages * L::kOperand);
#pragma unroll
          for (int k = 0; k < 8; ++k)
            mma_tensor(output, scores + k * 8, v + (k * 2048 >> 4), kInstruction<D, true>, i > 1 || k > 0);
          if (g == groups - 1) commit(&sh->v_empty[before % kStages]);
          if (i == tiles) commit(&sh->o_full[g]);
        }
        if (i < tiles) {
          if (!bar_wait(&sh->k_full[now % kStages], now / kStages & 1, &sh->abort)) return;
          if (i == 0) {
            uint32_t& t = g == 0 ? segment[0] : segment[1];
            if (!bar_wait(&sh->q_full[g], t & 1, &sh->abort)) return;
            ++t;
          }
          tensor_fence_after();
          const uint64_t q = row_descriptor(base + L::kQ + g * L::kOperand);
          const uint64_t keys = row_descriptor(base + L::kK + now % kStages * L::kOperand);
#pragma unroll
          for (int k = 0; k < D / 16; ++k) {
            const uint32_t at = ((k / 4) * 16384 + (k % 4) * 32) >> 4;
            mma_shared(scores, q + at, keys + at, kInstruction<128, false>, k > 0);
          }
          commit(&sh->s_full[g]);
          if (g == groups - 1) commit(&sh->k_empty[now % kStages]);
        }
      }
    }
    count += tiles;
  }
}

// --- warps 0-7 -------------------------------------------------------------

// Scores behind the row's last key, or of groups without a page, become -inf.
__device__ __forceinline__ void mask_scores(uint32_t scores_at, int seen, uint32_t absent) {
#pragma unroll 1
  for (int c = 0; c < 4; ++c) {
    float s[32];
    load_begin(s, scores_at + 32 * c);
    load_end(s);
#pragma unroll
    for (int i = 0; i < 32; ++i)
      if (32 * c + i >= seen || (absent >> (2 * c + i / 16) & 1)) s[i] = __uint_as_float(kNegInf);
    tensor_store32(scores_at + 32 * c, s);
  }
  tensor_wait_stores();
}

// Two at a time: the fp32 pairs of sm_100 take one issue slot.
__device__ __forceinline__ float2 exp2_pair(float x, float y, float f, float bias) {
  uint64_t r;
  asm("{\n\t.reg .b64 x, f, b;\n\tmov.b64 x, {%1, %2};\n\tmov.b64 f, {%3, %3};\n\tmov.b64 b, {%4, %4};\n\t"
      "fma.rn.f32x2 %0, x, f, b;\n\t}"
      : "=l"(r)
      : "f"(x), "f"(y), "f"(f), "f"(bias));
  return make_float2(exp2_fast(__uint_as_float((uint32_t)r)), exp2_fast(__uint_as_float((uint32_t)(r >> 32))));
}
__device__ __forceinline__ float2 add_pair(float2 a, float2 b) {
  uint64_t r;
  asm("{\n\t.reg .b64 x, y;\n\tmov.b64 x, {%1, %2};\n\tmov.b64 y, {%3, %4};\n\tadd.rn.f32x2 %0, x, y;\n\t}"
      : "=l"(r)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return make_float2(__uint_as_float((uint32_t)r), __uint_as_float((uint32_t)(r >> 32)));
}

// --- warps 0-7 -------------------------------------------------------------

template <int D>
__device__ __forceinline__ void softmax_role(const Args& a, Shared* sh, uint8_t* smem) {
  using L = Layout<D>;
  const int g = threadIdx.x / 128, r = threadIdx.x % 128;
  const uint32_t base = smem_of(smem);
  const uint32_t lanes = (uint32_t)(r / 32 * 32) << 16;
  const uint32_t scores_at = sh->tmem + lanes + kScoresAt + g * kGroupColumns;
  const uint32_t output_at = sh->tmem + lanes + kOutputsAt + g * kGroupColumns;
  const uint32_t q_at = base + L::kQ + g * L::kOperand;
  uint32_t count = 0, turn = 0, segment = 0;
  for (uint32_t n = 0;; ++n) {
    const Work* work = take_work(sh, n);
    if (__any_sync(0xFFFFFFFFu, work == nullptr)) return;
    const int begin = work->begin, end = work->end;
    if (g >= work->groups()) {
      count += end - begin;
      __syncwarp();
      if (threadIdx.x % 32 == 0) return_work(sh, n);
      continue;
    }
    const int at = work->first_row + g * kGroupRows + r;  // this thread's packed row
    const bool real = g * kGroupRows + r < work->rows;
    const int limit = real ? max(0, work->offset + at / a.group + 1) : 0;  // keys that it sees
    float factor;
    {  // q: one row a thread, scaled to an amax of 2^14..2^15
      const uint8_t* from = a.q + (work->start + at / a.group) * a.q_stride +
                            (int64_t)(work->head * a.group + at % a.group) * D * 2;
      const uint32_t infinite = a.bf16 ? 0x7F80u : 0x7C00u;
      uint32_t most = 0;  // magnitude bits of the largest finite value
#pragma unroll 4
      for (int c = 0; c < D / 8; ++c) {
        const uint4 v = real ? __ldg(reinterpret_cast<const uint4*>(from) + c) : make_uint4(0, 0, 0, 0);
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t lo = w[i] & 0x7FFFu, hi = w[i] >> 16 & 0x7FFFu;
          most = max(most, max(lo < infinite ? lo : 0u, hi < infinite ? hi : 0u));
        }
      }
      const uint32_t bits = __float_as_uint(unpack(a.bf16, most).x);
      const int e = bits == 0 ? 0 : min(14 - ((int)(bits >> 23) - 127), 100);
      const float up = __uint_as_float((uint32_t)(127 + e) << 23);
      factor = a.scale_log2 * __uint_as_float((uint32_t)(127 - e) << 23);
#pragma unroll 4
      for (int c = 0; c < D / 8; ++c) {
        const uint4 v = real ? __ldg(reinterpret_cast<const uint4*>(from) + c) : make_uint4(0, 0, 0, 0);
        const float2 x0 = unpack(a.bf16, v.x), x1 = unpack(a.bf16, v.y);
        const float2 x2 = unpack(a.bf16, v.z), x3 = unpack(a.bf16, v.w);
        store_shared(q_at + operand_at<D>(r, c),
                     make_uint4(pack_half(x0.x * up, x0.y * up), pack_half(x1.x * up, x1.y * up),
                                pack_half(x2.x * up, x2.y * up), pack_half(x3.x * up, x3.y * up)));
      }
      async_fence();
      tensor_fence_before();
      bar_arrive(&sh->q_full[g]);
    }
    float m = __uint_as_float(kNegInf), l = 0.0f, ref = -200.0f;  // ref: log2 of the largest V scale
    uint32_t nan[D / 32];
#pragma unroll
    for (int i = 0; i < D / 32; ++i) nan[i] = 0;

#pragma unroll 1
    for (int tile = begin; tile < end; ++tile, ++count) {
      if (!warp_wait(&sh->scale_full[count % kScaleRing], count / kScaleRing & 1, &sh->abort)) return;
      const Scales& scales = sh->scales[count % kScaleRing];
      float f[8];
#pragma unroll
      for (int b = 0; b < 8; ++b)  // a scale of zero must not meet a masked score's infinity
        f[b] = fmaxf(scales.k[b] * factor, 1e-37f);
      const float largest = scales.largest;
      const uint32_t absent = scales.absent;
      const int seen = limit - tile * kKeyTile;  // of this tile's keys
      const bool masked = __any_sync(0xFFFFFFFFu, seen < kKeyTile) || absent != 0;
      if (!warp_wait(&sh->s_full[g], turn & 1, &sh->abort)) return;
      ++turn;
      tensor_fence_after();
      if (masked) mask_scores(scores_at, seen, absent);

      // The row's maximum; then its scores again, which costs less than the
      // registers to keep them.
      float buffer[2][32];
      float most = __uint_as_float(kNegInf);
      load_begin(buffer[0], scores_at);
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        float(&s)[32] = buffer[c % 2];
        load_end(s);
        load_begin(buffer[(c + 1) % 2], scores_at + (c + 1) % 4 * 32);
        float top[4] = {s[0], s[1], s[16], s[17]};
#pragma unroll
        for (int i = 2; i < 16; i += 2) {
          top[0] = fmaxf(top[0], s[i]), top[1] = fmaxf(top[1], s[i + 1]);
          top[2] = fmaxf(top[2], s[16 + i]), top[3] = fmaxf(top[3], s[17 + i]);
        }
        most = fmaxf(most, fmaxf(fmaxf(top[0], top[1]) * f[2 * c], fmaxf(top[2], top[3]) * f[2 * c + 1]));
      }
      load_end(buffer[0]);
      if (__any_sync(0xFFFFFFFFu, most > m + kRaise || largest > ref)) {
        const float top = fmaxf(m, most);
        const float keep_l = top == m ? 1.0f : exp2_fast(m - top);
        if (tile != begin) {
          const float keep = keep_l * exp2_fast(ref - largest);
#pragma unroll 1
          for (int c = 0; c < D / 8; ++c) tensor_scale8(output_at + 8 * c, keep);
        }
        l *= keep_l;
        m = top;
        ref = largest;
      }
      const float shift = m == __uint_as_float(kNegInf) ? 0.0f : m;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        float(&s)[32] = buffer[c % 2];
        if (c > 0) load_end(s);
        if (c < 3) load_begin(buffer[(c + 1) % 2], scores_at + (c + 1) * 32);
        uint32_t p[16];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const int b = 2 * c + k;
          const float bias = scales.shift[b] - shift;
          float2 sum0 = make_float2(0.0f, 0.0f), sum1 = sum0;
#pragma unroll
          for (int i = 0; i < 16; i += 4) {
            const float2 x = exp2_pair(s[16 * k + i], s[16 * k + i + 1], f[b], bias);
            const float2 y = exp2_pair(s[16 * k + i + 2], s[16 * k + i + 3], f[b], bias);
            sum0 = add_pair(sum0, x);
            sum1 = add_pair(sum1, y);
            p[8 * k + i / 2] = pack_half(x.x, x.y);
            p[8 * k + i / 2 + 1] = pack_half(y.x, y.y);
          }
          sum0 = add_pair(sum0, sum1);
          l = fmaf(sum0.x + sum0.y, scales.inverse[b], l);
        }
        // P takes the columns of scores that have been read: 16 for these 32.
        tensor_store16(scores_at + 16 * c, p);
      }
      if (work->mixed(tile)) {
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
    const bool whole = work->slot < 0;
    const float scale = exp2_fast(ref - kWeightLog2) * (whole ? (l == 0.0f ? 0.0f : 1.0f / l) : 1.0f);
    float* slot = whole ? nullptr : a.partial + ((int64_t)blockIdx.x * 2 + work->slot) * slot_floats(a.rows, D);
    const int row = g * kGroupRows + r;
#pragma unroll
    for (int c = 0; c < D / 32; ++c) {
      float o[32];
      __syncwarp();
      load_begin(o, output_at + 32 * c);
      load_end(o);
#pragma unroll
      for (int i = 0; i < 32; ++i) o[i] = (nan[c] >> i & 1) != 0 ? __uint_as_float(0x7FC00000u) : o[i] * scale;
      if (whole) {  // through the tile of q, which is not read any more
#pragma unroll
        for (int k = 0; k < 4; ++k)
          store_shared(q_at + operand_at<D>(r, 4 * c + k),
                       make_uint4(pack_out(a, o[8 * k], o[8 * k + 1]), pack_out(a, o[8 * k + 2], o[8 * k + 3]),
                                  pack_out(a, o[8 * k + 4], o[8 * k + 5]), pack_out(a, o[8 * k + 6], o[8 * k + 7])));
      } else if (real) {
        float4* to = reinterpret_cast<float4*>(slot + (int64_t)row * D + 32 * c);
#pragma unroll
        for (int i = 0; i < 8; ++i)
          to[i] = make_float4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
      }
    }
    __syncwarp();
    if (whole) {  // the warp's 32 rows, D / 8 threads to a row
      const int first_row = g * kGroupRows + r / 32 * 32;
#pragma unroll 2
      for (int i = threadIdx.x % 32; i < 32 * (D / 8); i += 32) {
        const int k = i / (D / 8), chunk = i % (D / 8);
        if (first_row + k < work->rows) {
          const int to = work->first_row + first_row + k;
          uint8_t* out = a.out + (work->start + to / a.group) * a.out_stride +
                         (int64_t)(work->head * a.group + to % a.group) * D * 2 + chunk * 16;
          const uint4 v = load_shared(q_at + operand_at<D>(r / 32 * 32 + k, chunk));
          if (a.wide_out) {
            *reinterpret_cast<uint4*>(out) = v;
          } else {
            reinterpret_cast<uint32_t*>(out)[0] = v.x, reinterpret_cast<uint32_t*>(out)[1] = v.y;
            reinterpret_cast<uint32_t*>(out)[2] = v.z, reinterpret_cast<uint32_t*>(out)[3] = v.w;
          }
        }
      }
      if (real) write_lse(a, work->start + at / a.group, work->head * a.group + at % a.group, m, l);
    } else if (real) {
      slot[(int64_t)a.rows * D + row] = m;
      slot[(int64_t)a.rows * D + a.rows + row] = l;
    }
    __syncwarp();
    if (threadIdx.x % 32 == 0) return_work(sh, n);
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
    for (int i = 0; i < kWorkRing; ++i) {
      bar_init(&sh.work_full[i], 1);
      bar_init(&sh.work_empty[i], 13);  // warps 0-11 and the issuing thread
    }
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
  Walk<kThreads> walk(a, &sh.walk);
  tensor_fence_before();
  __syncthreads();
  tensor_fence_after();

  if (warp < 8) {
    more_registers<kSoftmaxRegisters>();
    softmax_role<D>(a, &sh, smem);
  } else if (warp < 12) {
    fewer_registers<kConvertRegisters>();
    convert_role<D>(a, &sh, smem);
  } else {
    fewer_registers<kIssueRegisters>();
    if (threadIdx.x == 12 * 32) {
      issue_role<D>(&sh, smem_of(smem));
      // Nothing of this CTA's is in flight when its tensor memory is freed.
      commit(&sh.drained);
      bool done = bar_try(&sh.drained, 0);
      for (int spins = 0; !done && spins < 1 << 20; ++spins) done = bar_try(&sh.drained, 0);
      if (!done) atomicOr(&g_extend_error, kErrExtendWaitTimeout);
    } else if (threadIdx.x == 13 * 32) {
      schedule_role(a, walk, &sh);
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
