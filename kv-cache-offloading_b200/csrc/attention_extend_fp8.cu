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
//   warps 8-11      K: cache -> registers -> f16 operand in shared memory
//   warps 12-15     V, in the same way
//   warps 16, 17    one thread issues the matrix products of row tile 0, of 1
//   warp 18         one thread walks the CTA's part of the work
//   warp 19         pages and scales of each key tile
//
// K, V and Q are f16 operands: e4m3 is a subset of f16, and q is scaled by a
// power of two to an amax of 2^14..2^15, where every bf16 value down to 2^-31
// of the row's largest is exact. The scores S = Q K^T are fp32 in tensor
// memory; a scale block is 16 tokens or more, so the scale of K enters once
// per 16 scores. P = 2^(x - m) takes the scale of V with it, as a fraction of
// 2^(n - m) (bias in the exponent), times 2^8, and goes back to tensor memory as
// the f16 operand of O += P V, in the place of its scores. n follows the largest
// x + log2(scale) that the row itself has met, so its terms keep their bits
// whatever scales other rows' keys have, or keys of no weight; it is kept as n - m,
// since m may be too large for a sum with it. Keys whose V is all
// zero do not count there: beside a large value, seen or not, a scale block holds
// little else. The sum of p is taken before that, per 16 keys, and divided by the
// same factor. m and n are raised only when they are passed by 6, so the
// accumulator is rescaled a few times in a row tile, not once in each key tile.
//
// Scores are made 64 keys at a time, in two sets of columns that take turns: the
// scores of half h + 1 are there when the softmax has done half h, so it does not
// wait for products. Rescaling O waits for the output of the half before.
//
// Measured: 2048 tokens over a history of 34816 keys, 32 / 8 heads of 128, in 1.40
// to 1.44 ms = 790 to 810 TFLOP/s, half of the rate of a plain f16 product. A
// softmax warp's chain of a half (wait, 64 scores out of tensor memory, maximum,
// exponentials, P back, arrival) takes 3000 cycles where the products of both
// row tiles take 1300. Without the exponentials the kernel took 8 % less,
// without the maximum too 12 %, without most of the products 6 %: it is the
// latency of the chain with two such warps to a scheduler that bounds it. An n
// for each row costs 2 to 4 % against one for the row tile, which lost a row's
// bits to keys that it does not see. Tried and slower: reading the scores while the half before is being weighed, one
// 128-key set of columns, all scores in registers at once, one thread that
// issues for both row tiles.
//
// Every wait is bounded; one that runs out sets an error flag that
// kvoff_device_error reads, and the kernel ends without waiting for anything but
// its own products. What roles read from one another may be torn or stale by then:
// it takes part in sums, but addresses, loop bounds and branches of a whole warp
// are made of what cannot be, or are checked. The scheduler leaves a record that
// has nothing to join.
#include "attention_fp8.h"
#include "codec.cuh"

namespace kvoff {
namespace attention {

__device__ int g_extend_error = 0;

namespace {

constexpr int kThreads = 640;
constexpr int kGroupRows = 128;    // rows of a tensor tile
constexpr int kStages = 2;         // of K and of V
constexpr int kTileRing = 4;       // pages and scales of a tile, ahead of K and V
constexpr int kWorkRing = 2;       // segments handed out ahead
constexpr float kRaise = 6.0f;     // log2 of how far P may pass 1
constexpr float kWeightLog2 = 8.0f;
constexpr float kLeastLog2 = -42.0f;  // of a V scale against 2^(n - m): P rounds to 0 in f16
constexpr uint32_t kNegInf = 0xFF800000u;
constexpr uint32_t kWaitNs = 1000;
constexpr uint32_t kTmemColumns = 512;
constexpr uint32_t kScoresAt = 0, kOutputsAt = 256, kGroupColumns = 128;
constexpr int kHalf = 64;           // keys of a step: half a key tile, half a row tile's columns

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

// A key tile's 16-key groups: where they are and their scales.
struct Tile {
  int64_t place[8];  // byte of the cache, at this head; negative: no page
  float k[8];
  float v[8];        // log2
  float most_v[2];   // of each half
  uint32_t absent;   // bit g: group g has no page
  int32_t run;       // all 128 keys are read and follow one another from place[0]
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
  uint64_t q_full[2];
  uint64_t s_full[2][2], p_full[2][2], o_done[2][2];  // of row tile and half
  uint64_t k_full[kStages], k_empty[kStages], v_full[kStages], v_empty[kStages];
  uint64_t tile_full[kTileRing];
  uint64_t drained[2];
  Tile tiles[kTileRing];
  uint32_t filled[kStages][8];  // of V's 16-key groups: four bits a byte, 0: the key is all zero
  uint32_t nan[kStages];  // n + 1: V of tile n, in this stage, holds NaN that some row must not meet
  uint32_t tmem;
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
// One arrival for a warp, after what all its lanes did: 128 of them would take
// their turns at the barrier.
__device__ __forceinline__ void warp_arrive(uint64_t* bar) {
  __syncwarp();
  if (threadIdx.x % 32 == 0) bar_arrive(bar);
}
// Waits for the phase of `parity`, at most `most` times kWaitNs. When that
// runs out the error flag is set and the thread goes on: what it computes then
// means nothing, but each later wait of its ends at its first look (`most` is 0),
// so the kernel ends, and no warp is torn apart on the way.
struct Patience {
  uint32_t most;
};
__device__ __forceinline__ void bar_wait(uint64_t* bar, uint32_t parity, Patience& patience) {
  uint32_t done;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t.reg .u32 n;\n\tmov.u32 n, 0;\n"
      "AGAIN:\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\t"
      "@p bra DONE;\n\t"
      "add.u32 n, n, 1;\n\t"
      "setp.lt.u32 q, n, %4;\n\t"
      "@q bra AGAIN;\n"
      "DONE:\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(done)
      : "r"(smem_of(bar)), "r"(parity), "r"(kWaitNs), "r"(patience.most)
      : "memory");
  if (done == 0) {
    if (patience.most != 0) atomicOr(&g_extend_error, kErrExtendWaitTimeout);
    patience.most = 0;
  }
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
// The upper word of a descriptor: 1024 bytes from 8 rows to the next 8, version,
// 128-byte swizzle.
constexpr uint32_t kDescriptorUp = 1024 >> 4 | 1u << 14 | 2u << 29;
// The lower word. K-major (the reduction runs along a row): the leading offset is
// not used. MN-major (it runs over rows): it leads from one 64-column block to
// the next.
__device__ __forceinline__ uint32_t row_descriptor(uint32_t address) { return 1u << 16 | address >> 4; }
__device__ __forceinline__ uint32_t column_descriptor(uint32_t address) {
  return (uint32_t)(16384 >> 4) << 16 | address >> 4;
}

// f16 operands, fp32 sums, M = 128; B is N x K along K, or along N.
template <int N, bool kBColumns>
constexpr uint32_t kInstruction = 1u << 4 | (kBColumns ? 1u << 16 : 0u) | (uint32_t)(N / 8) << 17 |
                                  (uint32_t)(128 / 16) << 24;

__device__ __forceinline__ void mma_shared(uint32_t d, uint32_t a, uint32_t b, uint32_t instruction,
                                           bool add) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 a, b;\n\tsetp.ne.u32 p, %4, 0;\n\t"
      "mov.b64 a, {%1, %5};\n\tmov.b64 b, {%2, %5};\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, p;\n\t}" ::"r"(d),
      "r"(a), "r"(b), "r"(instruction), "r"((uint32_t)add), "r"(kDescriptorUp)
      : "memory");
}
__device__ __forceinline__ void mma_tensor(uint32_t d, uint32_t a, uint32_t b, uint32_t instruction,
                                           bool add) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 b;\n\tsetp.ne.u32 p, %4, 0;\n\t"
      "mov.b64 b, {%2, %5};\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %3, p;\n\t}" ::"r"(d),
      "r"(a), "r"(b), "r"(instruction), "r"((uint32_t)add), "r"(kDescriptorUp)
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
// 640 threads are launched with 96 registers each; the shares of the five
// warpgroups add up to 5 * 96.
constexpr int kLaunchRegisters = 96, kSoftmaxRegisters = 136, kConvertRegisters = 72, kOtherRegisters = 64;
static_assert(2 * kSoftmaxRegisters + 2 * kConvertRegisters + kOtherRegisters == 5 * kLaunchRegisters, "registers");

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

// The next segment, or null (also when a wait has run out).
__device__ __forceinline__ const Work* take_work(Shared* sh, uint32_t n, Patience& patience) {
  const Work* work = &sh->work[n % kWorkRing];
  bar_wait(&sh->work_full[n % kWorkRing], n / kWorkRing & 1, patience);
  return patience.most == 0 || work->end < 0 ? nullptr : work;
}
__device__ __forceinline__ void return_work(Shared* sh, uint32_t n) { bar_arrive(&sh->work_empty[n % kWorkRing]); }

// --- warp 18 ---------------------------------------------------------------

__device__ __forceinline__ void schedule_role(const Args& a, Walk<kThreads>& walk, Shared* sh) {
  Patience patience{a.most_waits};
  uint32_t n = 0;
  Segment seg;
  for (bool more = true; more; ++n) {
    more = walk.next(a, &seg);
    bar_wait(&sh->work_empty[n % kWorkRing], (n / kWorkRing & 1) ^ 1, patience);
    if (patience.most == 0) {
      walk.give_up(a);
      return;
    }
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

// --- warps 8-15 ------------------------------------------------------------

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
  int t;  // thread of the warpgroup

  // Chunk and first row of this thread. Eight threads have four chunks of an
  // even row and of the next one, whose swizzled places in shared memory are
  // all different.
  __device__ __forceinline__ int chunk() const { return D == 128 ? t % 4 + t / 8 % 2 * 4 : t % 4; }
  __device__ __forceinline__ int row0() const { return D == 128 ? t / 32 * 4 + t / 16 % 2 * 2 + t / 4 % 2 : t / 4; }
  __device__ __forceinline__ int row(int i) const { return row0() + kRowsAPass * i; }

  // Where this thread reads in a group that begins at byte 0 of the cache.
  __device__ __forceinline__ int64_t from(int64_t row_bytes) const {
    return row0() % 16 * row_bytes + chunk() * 16;
  }
  // The rows of a tile that stand below `left`, zeros for the others.
  __device__ __forceinline__ void load(const uint8_t* cache, const Tile& tile, int left, uint4 (&raw)[kPasses]) const {
    const int64_t row_bytes = (int64_t)a.kv_heads * D;
    const int64_t first = tile.place[0];
    if (tile.run && first >= 0) {  // the page holds 128 rows from any tile's first on
      const uint8_t* at = cache + first + row0() * row_bytes + chunk() * 16;
#pragma unroll
      for (int i = 0; i < kPasses; ++i) {
        raw[i] = load_global(at);
        at += kRowsAPass * row_bytes;
      }
    } else {
      const uint8_t* at = cache + row0() % 16 * row_bytes + chunk() * 16;
#pragma unroll
      for (int i = 0; i < kPasses; ++i) {
        const int64_t group = tile.place[row(i) / 16];
        raw[i] = make_uint4(0, 0, 0, 0);
        if (row(i) < left && group >= 0) raw[i] = load_global(at + group);
      }
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

  // Notes the keys with a value that is not zero. A warp has 4 keys of each group, or
  // 8 of every other one (D = 64), and all their chunks.
  __device__ __forceinline__ void note_filled(int stage, const uint4 (&raw)[kPasses]) const {
    const int lane = t % 32, warp = t / 32;
    uint32_t mine = 0;  // of pass `lane`: the threads whose chunk is not zero
#pragma unroll
    for (int i = 0; i < kPasses; ++i) {
      const uint32_t any = (raw[i].x | raw[i].y | raw[i].z | raw[i].w) & 0x7F7F7F7Fu;
      const uint32_t mask = __ballot_sync(0xFFFFFFFFu, any != 0);
      if (lane == i) mine = mask;
    }
    if (lane >= kPasses) return;
    if (D == 128) {
      const uint32_t keys = ((mine & 0x0F0Fu) != 0 ? 1 : 0) | ((mine & 0xF0F0u) != 0 ? 2 : 0) |
                            ((mine & 0x0F0F0000u) != 0 ? 4 : 0) | ((mine & 0xF0F00000u) != 0 ? 8 : 0);
      reinterpret_cast<uint8_t*>(&sh->filled[stage][lane])[warp] = (uint8_t)keys;
    } else {
      uint32_t keys = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if ((mine >> 4 * i & 0xFu) != 0) keys |= 1u << (i + i / 4 * 4);
      reinterpret_cast<uint16_t*>(&sh->filled[stage][2 * lane + warp / 2])[warp % 2] = (uint16_t)keys;
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

// K and V run the same code: what the roles execute in each tile has to stay in the
// instruction cache together.
template <int D>
__device__ __forceinline__ void convert_role(const Args& a, Shared* sh, uint8_t* smem, bool is_v) {
  using L = Layout<D>;
  constexpr int kPasses = Convert<D>::kPasses;
  Convert<D> c{a, sh, (int)threadIdx.x % 128};
  const uint32_t operand = smem_of(smem) + (is_v ? L::kV : L::kK);
  const uint8_t* cache = is_v ? a.cache[1] : a.cache[0];
  uint64_t* full = is_v ? sh->v_full : sh->k_full;
  uint64_t* empty = is_v ? sh->v_empty : sh->k_empty;
  Patience patience{a.most_waits};
  uint32_t count = 0;  // key tiles so far, over all segments
  for (uint32_t n = 0;; ++n) {
    const Work* work = take_work(sh, n, patience);
    if (__any_sync(0xFFFFFFFFu, work == nullptr)) return;
    const int begin = work->begin, end = work->end, keys = work->keys;
    uint4 raw[kPasses];
    // Tile `tile` is put into shared memory, then tile + 1 is loaded: loads in
    // flight would be waited for by the fence and the arrival.
#pragma unroll 1
    for (int tile = begin - 1; tile < end; ++tile) {
      if (tile >= begin) {
        const int stage = count % kStages;
        bar_wait(&empty[stage], (count / kStages & 1) ^ 1, patience);
        if (is_v) c.note_filled(stage, raw);
        if (is_v && work->mixed(tile)) c.take_nan(stage, count, raw, smem + L::kNan + stage * L::kNanBytes);
        c.put(operand + stage * L::kOperand, raw);
        async_fence();
        warp_arrive(&full[stage]);
        ++count;
      }
      if (tile + 1 < end) {
        bar_wait(&sh->tile_full[count % kTileRing], count / kTileRing & 1, patience);
        if (patience.most != 0)  // else the entry may be anything
          c.load(cache, sh->tiles[count % kTileRing], keys - (tile + 1) * kKeyTile, raw);
      }
    }
    __syncwarp();
    if (threadIdx.x % 32 == 0) return_work(sh, n);
  }
}

// --- warp 19 ---------------------------------------------------------------

// Lane g < 8 has 16-key group g of each tile. Entry n + 4 of the ring is written
// when the scores of tile n + 2 are complete: they were issued after the output
// of tile n + 1, so the softmax of tile n is done with its scales, and K and V of
// tile n are loaded.
template <int D>
__device__ __forceinline__ void tile_role(const Args& a, Shared* sh) {
  const int lane = threadIdx.x % 32;
  const int blocks = a.page / 16 / a.block_tiles;  // scale blocks of a page
  const bool long_pages = a.page % kKeyTile == 0;
  Patience patience{a.most_waits};
  uint32_t count = 0;
  for (uint32_t n = 0;; ++n) {
    const Work* work = take_work(sh, n, patience);
    if (__any_sync(0xFFFFFFFFu, work == nullptr)) return;
    const int32_t* table = a.tables + work->seq * a.table_stride;
    const int begin = work->begin, end = work->end, keys = work->keys, head = work->head;
    auto page_of = [&](int tile) {  // checked when it is used, a tile later
      const int key = tile * kKeyTile + lane * 16;
      return lane < 8 && tile < end && key < keys ? __ldg(table + page_index(a, key)) : -1;
    };
    int page_next = page_of(begin);
#pragma unroll 1
    for (int tile = begin; tile < end; ++tile, ++count) {
      const int page = page_next < a.num_pages ? page_next : -1;
      page_next = page_of(tile + 1);
      int64_t place = -1;
      float k_scale = 0.0f, v_scale = 0.0f;
      if (page >= 0) {
        const int key = tile * kKeyTile + lane * 16, in_page = key - page_index(a, key) * a.page;
        place = (((int64_t)page * a.page + in_page) * a.kv_heads + head) * D;
        const int64_t at = ((int64_t)page * blocks + in_page / 16 / a.block_tiles) * a.kv_heads + head;
        k_scale = __ldg(a.scale[0] + at);
        v_scale = __ldg(a.scale[1] + at);
      }
      const uint32_t absent = __ballot_sync(0xFFFFFFFFu, page < 0) & 0xFFu;
      const float v_log2 = scale_log2_of(v_scale);
      float most = v_log2;  // of the half's four lanes
      most = fmaxf(most, __shfl_xor_sync(0xFFFFFFFFu, most, 1));
      most = fmaxf(most, __shfl_xor_sync(0xFFFFFFFFu, most, 2));
      if (count >= 2) {  // each phase in turn: a wait tells the last two apart only
        const uint32_t scores = count - 2;
        bar_wait(&sh->k_empty[scores % kStages], scores / kStages & 1, patience);
        if (__any_sync(0xFFFFFFFFu, patience.most == 0)) return;  // the entry may still be read
      }
      Tile& t = sh->tiles[count % kTileRing];
      if (lane < 8) {
        t.place[lane] = place;
        t.k[lane] = k_scale;
        t.v[lane] = v_log2;
        if (lane % 4 == 0) t.most_v[lane / 4] = most;
      }
      if (lane == 0) {
        t.absent = absent;
        t.run = long_pages && keys - tile * kKeyTile >= kKeyTile && absent == 0;
      }
      __syncwarp();
      if (lane == 0) bar_arrive(&sh->tile_full[count % kTileRing]);
    }
    __syncwarp();
    if (lane == 0) return_work(sh, n);
  }
}

// --- warps 16, 17 ----------------------------------------------------------

// One thread for each 128-row tile g.
template <int D>
__device__ __forceinline__ void issue_role(const Args& a, Shared* sh, uint32_t base, int g) {
  using L = Layout<D>;
  const uint32_t scores = sh->tmem + kScoresAt + g * kGroupColumns, output = sh->tmem + kOutputsAt + g * kGroupColumns;
  const uint32_t q = row_descriptor(base + L::kQ + g * L::kOperand);
  const uint32_t k0 = row_descriptor(base + L::kK), v0 = column_descriptor(base + L::kV);
  Patience patience{a.most_waits};
  uint32_t count = 0, turn = 0, segment = 0;  // key tiles so far, of the CTA and of this row tile
  for (uint32_t n = 0;; ++n) {
    const Work* work = take_work(sh, n, patience);
    if (work == nullptr) return;
    const int tiles = work->end - work->begin;
    const bool idle = g >= work->groups();
    return_work(sh, n);
    if (idle) {  // K and V are not read, but given back in their order
      for (int i = 0; i < tiles; ++i, ++count) {
        const uint32_t stage = count % kStages, parity = count / kStages & 1;
        bar_wait(&sh->k_full[stage], parity, patience);
        bar_arrive(&sh->k_empty[stage]);
        bar_wait(&sh->v_full[stage], parity, patience);
        bar_arrive(&sh->v_empty[stage]);
      }
      continue;
    }
    bar_wait(&sh->q_full[g], segment & 1, patience);
    ++segment;
    // Step h: the output of half h - 2, then the scores of half h in its columns.
#pragma unroll 1
    for (int h = 0; h < 2 * tiles + 2; ++h) {
      const uint32_t half = h & 1;
      if (h >= 2) {
        const uint32_t tile = count + (h - 2) / 2, stage = tile % kStages;
        const uint32_t v = v0 + stage * (L::kOperand >> 4) + half * (kHalf * 128 >> 4);
        if (half == 0) bar_wait(&sh->v_full[stage], tile / kStages & 1, patience);
        bar_wait(&sh->p_full[g][half], turn & 1, patience);
        turn += half;
        tensor_fence_after();
#pragma unroll
        for (int k = 0; k < kHalf / 16; ++k)
          mma_tensor(output, scores + half * kHalf + k * 8, v + (k * 2048 >> 4), kInstruction<D, true>, h > 2 || k > 0);
        commit(&sh->o_done[g][half]);
        if (half == 1) commit(&sh->v_empty[stage]);
      }
      if (h < 2 * tiles) {
        const uint32_t tile = count + h / 2, stage = tile % kStages;
        const uint32_t keys = k0 + stage * (L::kOperand >> 4) + half * (kHalf * 128 >> 4);
        if (half == 0) bar_wait(&sh->k_full[stage], tile / kStages & 1, patience);
        tensor_fence_after();
#pragma unroll
        for (int k = 0; k < D / 16; ++k) {
          const uint32_t at = ((k / 4) * 16384 + (k % 4) * 32) >> 4;
          mma_shared(scores + half * kHalf, q + at, keys + at, kInstruction<kHalf, false>, k > 0);
        }
        commit(&sh->s_full[g][half]);
        if (half == 1) commit(&sh->k_empty[stage]);
      }
    }
    count += tiles;
  }
}

// Scores of a half behind the row's last key, or of groups without a page,
// become -inf. `seen`, `absent`: of this half.
__device__ __forceinline__ void mask_scores(uint32_t scores_at, int seen, uint32_t absent) {
#pragma unroll 1
  for (int c = 0; c < kHalf / 32; ++c) {
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

// Log2 units of a raw score of group b. A scale of zero must not meet a masked
// score's infinity.
__device__ __forceinline__ float factor_of(const Tile& scales, int b, float factor) {
  return fmaxf(scales.k[b] * factor, 1e-37f);
}

// The largest scores of the two groups of chunk c, in log2 units.
__device__ __forceinline__ void top_of(const float (&s)[32], const Tile& scales, int c, float factor, float* most) {
  float top[4] = {s[0], s[1], s[16], s[17]};
#pragma unroll
  for (int i = 2; i < 16; i += 2) {
    top[0] = fmaxf(top[0], s[i]), top[1] = fmaxf(top[1], s[i + 1]);
    top[2] = fmaxf(top[2], s[16 + i]), top[3] = fmaxf(top[3], s[17 + i]);
  }
  most[0] = fmaxf(top[0], top[1]) * factor_of(scales, 2 * c, factor);
  most[1] = fmaxf(top[2], top[3]) * factor_of(scales, 2 * c + 1, factor);
}

__device__ __forceinline__ float largest_of(const float (&x)[4]) { return fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])); }

// The largest of the four groups' scores with their V scales, against m.
__device__ __forceinline__ float term_of(const float (&x)[4], const float (&v)[4], float m) {
  return fmaxf(fmaxf((x[0] - m) + v[0], (x[1] - m) + v[1]), fmaxf((x[2] - m) + v[2], (x[3] - m) + v[3]));
}

// P of the 32 scores of chunk c; its sums go into l. P takes the columns of
// scores that have been read: 16 for these 32. `v`: V scales of the two groups,
// `unit`: n - m. The bias is rounded like a score, for P and its sum alike.
__device__ __forceinline__ void weigh(const float (&s)[32], const Tile& scales, int c, float factor, float m,
                                      float unit, const float* v, uint32_t scores_at, float& l) {
  uint32_t p[16];
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const int b = 2 * c + k;
    const float f = factor_of(scales, b, factor), fraction = v[k] - unit;
    const float shift = (fraction < kLeastLog2 ? kLeastLog2 : fraction) + kWeightLog2, bias = shift - m;
    float2 sum0 = make_float2(0.0f, 0.0f), sum1 = sum0;
#pragma unroll
    for (int i = 0; i < 16; i += 4) {
      const float2 x = exp2_pair(s[16 * k + i], s[16 * k + i + 1], f, bias);
      const float2 y = exp2_pair(s[16 * k + i + 2], s[16 * k + i + 3], f, bias);
      sum0 = add_pair(sum0, x);
      sum1 = add_pair(sum1, y);
      p[8 * k + i / 2] = pack_half(x.x, x.y);
      p[8 * k + i / 2 + 1] = pack_half(y.x, y.y);
    }
    sum0 = add_pair(sum0, sum1);
    l = fmaf(sum0.x + sum0.y, exp2_fast(-shift), l);
  }
  tensor_store16(scores_at + 16 * (c % 2), p);
}

// Which of the 32 keys of chunk c are not all zero in V.
__device__ __forceinline__ uint32_t filled_of(const uint32_t* filled, int c) {
  uint32_t keys = 0;
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const uint32_t w = filled[2 * c + k];
    keys |= (w & 0xFu | w >> 4 & 0xF0u | w >> 8 & 0xF00u | w >> 12 & 0xF000u) << 16 * k;
  }
  return keys;
}

// Adds the weights of chunk c's other keys to l, and takes the keys out: they add
// nothing to O, and P with their scale may not fit f16.
__device__ __forceinline__ void set_aside(float (&s)[32], const Tile& scales, int c, float factor, float m,
                                          uint32_t filled, float& l) {
#pragma unroll
  for (int i = 0; i < 32; ++i)
    if ((filled >> i & 1) == 0) {
      l += exp2_fast(fmaf(s[i], factor_of(scales, 2 * c + i / 16, factor), -m));
      s[i] = __uint_as_float(kNegInf);
    }
}

template <int D>
__device__ __forceinline__ void softmax_role(const Args& a, Shared* sh, uint8_t* smem) {
  using L = Layout<D>;
  const int g = threadIdx.x / 128, r = threadIdx.x % 128;
  const uint32_t base = smem_of(smem);
  const uint32_t lanes = (uint32_t)(r / 32 * 32) << 16;
  const uint32_t scores_at = sh->tmem + lanes + kScoresAt + g * kGroupColumns;
  const uint32_t output_at = sh->tmem + lanes + kOutputsAt + g * kGroupColumns;
  const uint32_t q_at = base + L::kQ + g * L::kOperand;
  Patience patience{a.most_waits};
  uint32_t count = 0, turn = 0;  // key tiles so far, of the CTA and of this row tile
  for (uint32_t n = 0;; ++n) {
    const Work* work = take_work(sh, n, patience);
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
      warp_arrive(&sh->q_full[g]);
    }
    // Largest x, and largest x + log2(V scale) against it; sum of 2^(x - m). `base` is m,
    // 0 for a row that has seen nothing.
    float m = __uint_as_float(kNegInf), unit = kZeroLog2, l = 0.0f, base = 0.0f;
    uint32_t nan[D / 32];
#pragma unroll
    for (int i = 0; i < D / 32; ++i) nan[i] = 0;

#pragma unroll 1
    for (int h = 2 * begin; h < 2 * end; ++h) {
      const int half = h & 1;
      const uint32_t half_at = scores_at + half * kHalf;
      // The scores first: a row tile that sat out segments may be ahead of the
      // ring of tiles by more than its barriers can tell.
      bar_wait(&sh->s_full[g][half], turn & 1, patience);
      tensor_fence_after();
      if (half == 0) bar_wait(&sh->tile_full[count % kTileRing], count / kTileRing & 1, patience);
      const Tile& scales = sh->tiles[count % kTileRing];
      const uint32_t absent = scales.absent >> 4 * half & 0xFu;
      const int seen = limit - h * kHalf;  // of this half's keys
      if (__any_sync(0xFFFFFFFFu, seen < kHalf || absent != 0)) mask_scores(half_at, seen, absent);
      float x[32], y[32];
      load_begin(x, half_at);
      load_begin(y, half_at + 32);
      load_end(x);
      load_end(y);
      float tops[4], v[4];
      top_of(x, scales, 2 * half, factor, tops);
      top_of(y, scales, 2 * half + 1, factor, tops + 2);
#pragma unroll
      for (int b = 0; b < 4; ++b) v[b] = scales.v[4 * half + b];
      const float most = largest_of(tops);
      if (__any_sync(0xFFFFFFFFu, most > __fadd_rd(m, fminf(kRaise, unit + kRaise - scales.most_v[half])))) {
        const int stage = count % kStages;
        bar_wait(&sh->v_full[stage], count / kStages & 1, patience);
        const uint32_t low = filled_of(sh->filled[stage], 2 * half), high = filled_of(sh->filled[stage], 2 * half + 1);
        const float top = fmaxf(m, most);
        if (top != m) l *= exp2_fast(m - top);
        base = top == __uint_as_float(kNegInf) ? 0.0f : top;
        if (__any_sync(0xFFFFFFFFu, (low & high) != 0xFFFFFFFFu)) {
          set_aside(x, scales, 2 * half, factor, base, low, l);
          set_aside(y, scales, 2 * half + 1, factor, base, high, l);
          top_of(x, scales, 2 * half, factor, tops);
          top_of(y, scales, 2 * half + 1, factor, tops + 2);
        }
        const float moved = top == __uint_as_float(kNegInf) ? kZeroLog2 : unit + (m - top);
        unit = fmaxf(fmaxf(moved, term_of(tops, v, top)), kZeroLog2);
        if (h != 2 * begin && __any_sync(0xFFFFFFFFu, unit != moved)) {
          // Not before the output of the half before is complete.
          bar_wait(&sh->o_done[g][half ^ 1], (turn - (half ^ 1)) & 1, patience);
          tensor_fence_after();
          const float keep = exp2_fast(moved - unit);
#pragma unroll 1
          for (int c = 0; c < D / 8; ++c) tensor_scale8(output_at + 8 * c, keep);
        }
        m = top;
      }
      weigh(x, scales, 2 * half, factor, base, unit, v, half_at, l);
      weigh(y, scales, 2 * half + 1, factor, base, unit, v + 2, half_at, l);
      if (work->mixed(h / 2)) {
        const int stage = count % kStages;
        bar_wait(&sh->v_full[stage], count / kStages & 1, patience);
        if (__any_sync(0xFFFFFFFFu, *reinterpret_cast<volatile uint32_t*>(&sh->nan[stage]) == count + 1)) {
          const uint32_t* masks = reinterpret_cast<const uint32_t*>(smem + L::kNan + stage * L::kNanBytes) +
                                  half * kHalf * (D / 32);
          for (int i = 0; i < min(seen, kHalf); ++i)
#pragma unroll
            for (int w = 0; w < D / 32; ++w) nan[w] |= masks[i * (D / 32) + w];
          __syncwarp();
        }
      }
      tensor_wait_stores();
      tensor_fence_before();
      warp_arrive(&sh->p_full[g][half]);
      turn += half;
      count += half;
    }

    bar_wait(&sh->o_done[g][1], (turn - 1) & 1, patience);
    tensor_fence_after();
    // 2^(n - m) may be as small as a scale can be; a row of zero scales is zero.
    const bool whole = work->slot < 0;
    const float scale = exp2_fast(unit - kWeightLog2) * (whole ? (l == 0.0f ? 0.0f : 1.0f / l) : 1.0f);
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
      bar_init(&sh.q_full[g], 4);  // one for each warp
      for (int h = 0; h < 2; ++h) {
        bar_init(&sh.s_full[g][h], 1);
        bar_init(&sh.p_full[g][h], 4);
        bar_init(&sh.o_done[g][h], 1);
      }
    }
    for (int i = 0; i < kStages; ++i) {
      bar_init(&sh.k_full[i], 4);
      bar_init(&sh.k_empty[i], 2);  // one for each row tile
      bar_init(&sh.v_full[i], 4);
      bar_init(&sh.v_empty[i], 2);
    }
    for (int i = 0; i < kTileRing; ++i) bar_init(&sh.tile_full[i], 1);
    for (int i = 0; i < kWorkRing; ++i) {
      bar_init(&sh.work_full[i], 1);
      bar_init(&sh.work_empty[i], 19);  // all warps but the scheduler
    }
    for (int g = 0; g < 2; ++g) bar_init(&sh.drained[g], 1);
    sh.nan[0] = sh.nan[1] = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 16) {
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
  } else if (warp < 16) {
    fewer_registers<kConvertRegisters>();
    convert_role<D>(a, &sh, smem, warp >= 12);
  } else {
    fewer_registers<kOtherRegisters>();
    if (warp < 18) {
      if (threadIdx.x % 32 == 0) {
        issue_role<D>(a, &sh, smem_of(smem), warp - 16);
        // Nothing of this CTA's is in flight when its tensor memory is freed.
        commit(&sh.drained[warp - 16]);
        Patience patience{kMostWaits};
        bar_wait(&sh.drained[warp - 16], 0, patience);
      }
    } else if (warp == 18) {
      if (threadIdx.x % 32 == 0) schedule_role(a, walk, &sh);
    } else {
      tile_role<D>(a, &sh);
    }
    __syncwarp();
  }
  if (!a.direct) launch_dependents();
  tensor_fence_before();
  __syncthreads();
  tensor_fence_after();
  if (warp == 16)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(sh.tmem), "r"(kTmemColumns));
}

template <int D>
int launch(const Args& a, int grid, cudaStream_t stream) {
  KVOFF_TRY(allow_shared<attention_extend_fp8_kernel<D>>(Layout<D>::kBytes));
  attention_extend_fp8_kernel<D><<<grid, kThreads, Layout<D>::kBytes, stream>>>(a);
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
