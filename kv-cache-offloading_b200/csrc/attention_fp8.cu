// Entry points of attention over the e4m3 paged cache, and the join of rows
// whose keys were read by several CTAs.
#include "attention_fp8.h"

#include <string.h>

namespace kvoff {
namespace attention {
namespace {

constexpr int kJoinThreads = 256;

// Every record's CTA joins the split row tile that begins in that CTA of the
// attention kernel: o = sum_c 2^(m_c - m) o_c / sum_c 2^(m_c - m) l_c over its
// parts, in the order of their keys, so the result does not depend on timing.
// A warp takes a row and blockIdx.y 64 values of it; lane i looks at part i, so
// that the parts' maxima and then their sums are read side by side.
__global__ void __launch_bounds__(kJoinThreads) join_kernel(const __grid_constant__ Args a, int dim) {
  asm volatile("griddepcontrol.wait;" ::: "memory");  // the parts are complete
  const int first = blockIdx.x;
  const Record record = a.records[first];
  if (record.further < 0) return;
  Sequence seq;
  seq.load(a, record.seq);
  const int rows = min(a.rows, seq.q_len * a.group - record.tile * a.rows);
  const int lane = threadIdx.x % 32, d = blockIdx.y * 64 + lane * 2;
  const int64_t slot = slot_floats(a.rows, dim);
  const float none = __int_as_float(0xFF800000);
  for (int row = threadIdx.x / 32 + blockIdx.z * (kJoinThreads / 32); row < rows;
       row += kJoinThreads / 32 * gridDim.z) {
    float most = none, l = 0.0f;
    float2 sum = make_float2(0.0f, 0.0f);
    bool any = false;
    for (int base = 0; base <= record.further; base += 32) {
      // Part 0 is the CTA's own (slot 1), part i continues it in CTA first + i * stride.
      const int part = base + lane, cta = first + part * a.stride;
      bool valid = false;
      if (part <= record.further) valid = part == 0 ? record.valid[1] != 0 : a.records[cta].valid[0] != 0;
      const float* p = a.partial + ((int64_t)cta * 2 + (part == 0 ? 1 : 0)) * slot;
      const float m = valid ? p[a.rows * dim + row] : none;
      const float part_l = valid ? p[a.rows * dim + a.rows + row] : 0.0f;
      float top = m;
#pragma unroll
      for (int k = 16; k > 0; k /= 2) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, k));
      top = fmaxf(top, most);
      // Without a key seen the sums are 0, or NaN from NaN scores: they are added.
      const float take = valid ? (top == none ? 1.0f : exp2_fast(m - top)) : 0.0f;
      const float keep = top == none || most == top ? 1.0f : exp2_fast(most - top);
      float add = take * part_l;
      if (!valid) add = 0.0f;
#pragma unroll
      for (int k = 16; k > 0; k /= 2) add += __shfl_xor_sync(0xFFFFFFFFu, add, k);
      l = l * keep + add;
      sum.x *= keep;
      sum.y *= keep;
      most = top;
      const uint32_t mask = __ballot_sync(0xFFFFFFFFu, valid);
      any = any || mask != 0;
      const int last = min(31, record.further - base);
#pragma unroll 8
      for (int i = 0; i <= last; ++i) {
        const float weight = __shfl_sync(0xFFFFFFFFu, take, i);
        if ((mask >> i & 1) != 0) {
          const int from = first + (base + i) * a.stride;
          const float2 x = *reinterpret_cast<const float2*>(
              a.partial + ((int64_t)from * 2 + (base + i == 0 ? 1 : 0)) * slot + row * dim + d);
          sum.x += weight * x.x;
          sum.y += weight * x.y;
        }
      }
    }
    if (!any) continue;  // one CTA had all of it and wrote the result
    const int at = record.tile * a.rows + row;
    const int token = seq.start + at / a.group, head = record.head * a.group + at % a.group;
    const float scale = l == 0.0f ? 0.0f : 1.0f / l;
    write_pair(a, token, head, dim, d, sum.x * scale, sum.y * scale);
    if (d == 0) write_lse(a, token, head, most, l);
  }
}

}  // namespace

int launch_join(const Args& a, int dim, int grid, cudaStream_t stream) {
  cudaLaunchConfig_t config{};
  config.gridDim = dim3(grid, dim / 64, a.rows > 32 ? 8 : 1);
  config.blockDim = dim3(kJoinThreads);
  config.stream = stream;
  cudaLaunchAttribute attribute[1];
  attribute[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attribute[0].val.programmaticStreamSerializationAllowed = 1;
  config.attrs = attribute;
  config.numAttrs = 1;
  return cuda_status(cudaLaunchKernelEx(&config, join_kernel, a, dim), "attention_fp8 join launch");
}

namespace {

// Longest context (in keys) that one CTA reads alone rather than sharing it:
// the join is a second launch. The host knows the tables' width and not the
// contexts, so short contexts behind wide tables are shared too (8 heads of 128,
// 300 keys: 1 sequence 7.4 us, with a table of 40960 keys 10.8; 4 sequences 7.6
// and 14.7).
constexpr int64_t kDirectKeys = 1024;

struct Shape {
  int64_t seqs, max_q, keys, q_heads, kv_heads, dim;
};

// How a call is launched: rows of a tile, CTAs, and whether rows are split.
struct Choice {
  int rows, grid, stride;
  int64_t max_tiles;
  bool direct, extend;
};

Choice choose(const Shape& s) {
  Choice c{};
  const int64_t rows = s.max_q * (s.q_heads / s.kv_heads);
  // The decode kernel reads the cache once for 16 rows, the prompt kernel once
  // for 256 and at the tensor cores' rate, but it takes longer to begin. Measured
  // (8 heads of 128, us, decode kernel / prompt kernel): 24 rows of 34816 keys 49
  // / 60, 32 rows 49 / 59, 64 rows 76 / 61; 64 rows of 300 keys 10.7 / 18.6.
  c.extend = rows > (s.keys <= kDirectKeys ? 64 : 32);
  c.rows = c.extend ? kExtendRows : rows <= 8 ? 8 : kDecodeRows;
  c.max_tiles = (rows + c.rows - 1) / c.rows;
  const int64_t ctas = s.seqs * s.kv_heads * c.max_tiles;
  c.direct = s.keys <= kDirectKeys && ctas <= 0x7FFFFFFFll;
  c.stride = c.extend ? 1 : (int)s.kv_heads;
  const int parts = sm_count() / (int)s.kv_heads;  // of a head's work
  c.grid = c.direct ? (int)ctas : c.extend ? sm_count() : (parts > 1 ? parts : 1) * c.stride;
  return c;
}

int64_t workspace_of(const Choice& c, int64_t dim) {
  if (c.direct) return 0;
  return c.grid * ((int64_t)sizeof(Record) + 2 * slot_floats(c.rows, (int)dim) * (int64_t)sizeof(float));
}

int check_shape(const Shape& s, int64_t page) {
  if (s.seqs < 0 || s.max_q < 0 || s.keys < 0 || s.q_heads <= 0 || s.kv_heads <= 0 || page <= 0)
    return fail(KVOFF_EINVAL, "kvoff_attention_fp8: bad sizes");
  if (s.dim != 64 && s.dim != 128)
    return fail(KVOFF_EINVAL, "kvoff_attention_fp8: head_dim %lld is not 64 or 128",
                (long long)s.dim);
  if (s.q_heads % s.kv_heads != 0 || s.q_heads > 65535)
    return fail(KVOFF_EINVAL, "kvoff_attention_fp8: %lld query heads do not divide over %lld KV heads",
                (long long)s.q_heads, (long long)s.kv_heads);
  if (page % 16 != 0)
    return fail(KVOFF_EINVAL, "kvoff_attention_fp8: page size %lld is not a multiple of 16",
                (long long)page);
  if (s.seqs > 0x7FFFFFFFll || s.keys > 0x7FFFFF00ll || s.max_q > 0x7FFFFFFFll / s.q_heads)
    return fail(KVOFF_EINVAL, "kvoff_attention_fp8: sizes exceed 32 bits");
  return KVOFF_OK;
}

}  // namespace
}  // namespace attention
}  // namespace kvoff

using namespace kvoff;

extern "C" int kvoff_attention_fp8_workspace(int64_t num_seqs, int64_t max_seqlen_q,
                                             int64_t table_width, int64_t page_size,
                                             int64_t q_heads, int64_t kv_heads, int64_t head_dim,
                                             int64_t* bytes) {
  if (bytes == nullptr) return fail(KVOFF_EINVAL, "kvoff_attention_fp8_workspace: null output");
  if (table_width < 0 || (page_size > 0 && table_width > 0x7FFFFF00ll / page_size))
    return fail(KVOFF_EINVAL, "kvoff_attention_fp8: sizes exceed 32 bits");
  const attention::Shape s{num_seqs, max_seqlen_q, table_width * page_size, q_heads, kv_heads, head_dim};
  KVOFF_TRY(attention::check_shape(s, page_size));
  *bytes = attention::workspace_of(attention::choose(s), head_dim);
  return ok();
}

extern "C" int kvoff_attention_fp8(
    const void* q, int64_t q_stride_bytes, void* out, int64_t out_stride_bytes, float* lse,
    const void* k_cache, const void* v_cache, const float* k_scale, const float* v_scale,
    int64_t num_pages, int64_t page_size, int64_t scale_block, const int32_t* block_tables,
    int64_t table_stride, int64_t table_width, const int32_t* context_lens,
    const int32_t* cu_seqlens_q, int64_t num_seqs, int64_t num_tokens, int64_t max_seqlen_q,
    int64_t q_heads, int64_t kv_heads, int64_t head_dim, int32_t dtype, float softmax_scale,
    void* workspace, int64_t workspace_bytes, void* stream) {
  if (injected("attention_fp8")) return KVOFF_EINJECTED;
  if (table_width < 0 || num_pages < 0 || num_pages > 0x7FFFFFFFll || num_tokens < 0 ||
      q_stride_bytes < 0 || out_stride_bytes < 0 || table_stride < 0 ||
      (page_size > 0 && table_width > 0x7FFFFF00ll / page_size))
    return fail(KVOFF_EINVAL, "kvoff_attention_fp8: bad sizes");
  const attention::Shape s{num_seqs, max_seqlen_q, table_width * page_size, q_heads, kv_heads, head_dim};
  KVOFF_TRY(attention::check_shape(s, page_size));
  if (scale_block < 16 || (scale_block & (scale_block - 1)) != 0 || page_size % scale_block != 0)
    return fail(KVOFF_EINVAL,
                "kvoff_attention_fp8: a scale block is 16 * 2^n tokens and divides the page of %lld",
                (long long)page_size);
  if (dtype != KVOFF_BF16 && dtype != KVOFF_FP16)
    return fail(KVOFF_EINVAL, "kvoff_attention_fp8: q and out are bf16 or fp16");
  if (cu_seqlens_q == nullptr && (num_tokens != num_seqs || max_seqlen_q != 1))
    return fail(KVOFF_EINVAL, "kvoff_attention_fp8: without cu_seqlens_q each sequence has one token");
  if (num_tokens > 0x7FFFF000ll / q_heads)
    return fail(KVOFF_EINVAL, "kvoff_attention_fp8: sizes exceed 32 bits");
  if (!(softmax_scale > 0.0f && softmax_scale < 3.4e38f))
    return fail(KVOFF_EINVAL, "kvoff_attention_fp8: softmax_scale must be positive and finite");
  if (num_seqs == 0 || num_tokens == 0) return ok();
  if (max_seqlen_q < 1)
    return fail(KVOFF_EINVAL, "kvoff_attention_fp8: max_seqlen_q %lld for %lld tokens",
                (long long)max_seqlen_q, (long long)num_tokens);
  if (q == nullptr || out == nullptr || context_lens == nullptr ||
      (s.keys > 0 && (k_cache == nullptr || v_cache == nullptr || k_scale == nullptr ||
                      v_scale == nullptr || block_tables == nullptr)))
    return fail(KVOFF_EINVAL, "kvoff_attention_fp8: null pointer");
  const uintptr_t wide = reinterpret_cast<uintptr_t>(q) | (uintptr_t)q_stride_bytes |
                         reinterpret_cast<uintptr_t>(k_cache) | reinterpret_cast<uintptr_t>(v_cache);
  const uintptr_t pairs = reinterpret_cast<uintptr_t>(out) | (uintptr_t)out_stride_bytes;
  if ((wide & 15u) != 0 || (pairs & 3u) != 0)
    return fail(KVOFF_EINVAL,
                "kvoff_attention_fp8: q and the caches must be 16-byte aligned, out 4-byte");
  if (num_tokens > 1 && out_stride_bytes < q_heads * head_dim * 2)
    return fail(KVOFF_EINVAL, "kvoff_attention_fp8: rows of the output overlap");
  const attention::Choice c = attention::choose(s);
  const int64_t need = attention::workspace_of(c, head_dim);
  if (need > 0 && (workspace == nullptr || workspace_bytes < need ||
                   (reinterpret_cast<uintptr_t>(workspace) & 15u) != 0))
    return fail(KVOFF_EINVAL, "kvoff_attention_fp8: needs a 16-byte aligned workspace of %lld bytes",
                (long long)need);
  attention::Args a{};
  a.q = static_cast<const uint8_t*>(q);
  a.out = static_cast<uint8_t*>(out);
  a.lse = lse;
  a.q_stride = q_stride_bytes;
  a.out_stride = out_stride_bytes;
  a.cache[0] = static_cast<const uint8_t*>(k_cache);
  a.cache[1] = static_cast<const uint8_t*>(v_cache);
  a.scale[0] = k_scale;
  a.scale[1] = v_scale;
  a.tables = block_tables;
  a.table_stride = table_stride;
  a.contexts = context_lens;
  a.starts = cu_seqlens_q;
  a.scale_log2 = softmax_scale * 1.4426950408889634f;
  a.table_width = (int32_t)table_width;
  a.num_pages = (int32_t)num_pages;
  a.page = (int32_t)page_size;
  a.block_tiles = (int32_t)(scale_block / 16);
  a.page_shift = -1;
  if ((page_size & (page_size - 1)) == 0)
    for (a.page_shift = 0; (1ll << a.page_shift) < page_size;) ++a.page_shift;
  a.seqs = (int32_t)num_seqs;
  a.num_tokens = (int32_t)num_tokens;
  a.q_heads = (int32_t)q_heads;
  a.kv_heads = (int32_t)kv_heads;
  a.group = (int32_t)(q_heads / kv_heads);
  a.rows = c.rows;
  while ((1 << a.row_shift) < c.rows) ++a.row_shift;
  a.tiles_per_cost = 1.0 / (attention::kKeyTile * (double)(q_heads / kv_heads));
  a.fixed = c.extend ? attention::kExtendFixed : attention::kDecodeFixed;
  a.max_tiles = (int32_t)c.max_tiles;
  a.direct = c.direct;
  a.stride = c.stride;
  a.bf16 = dtype == KVOFF_BF16;
  a.wide_out = (pairs & 15u) == 0;
  a.most_waits = c.extend && injected("attention_wait") ? 1 : attention::kMostWaits;
  a.records = static_cast<attention::Record*>(workspace);
  a.partial = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) +
                                       c.grid * (int64_t)sizeof(attention::Record));
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  KVOFF_TRY(c.extend ? attention::launch_extend(a, (int)head_dim, c.grid, st)
                     : attention::launch_decode(a, (int)head_dim, c.grid, st));
  if (!c.direct) KVOFF_TRY(attention::launch_join(a, (int)head_dim, c.grid, st));
  return ok();
}

extern "C" int kvoff_attention_fp8_packed(const int64_t* a) {
  if (a == nullptr) return fail(KVOFF_EINVAL, "kvoff_attention_fp8_packed: null pointer");
  double softmax_scale;
  memcpy(&softmax_scale, a + 24, sizeof(softmax_scale));
  return kvoff_attention_fp8(
      reinterpret_cast<const void*>(a[0]), a[1], reinterpret_cast<void*>(a[2]), a[3],
      reinterpret_cast<float*>(a[4]), reinterpret_cast<const void*>(a[5]),
      reinterpret_cast<const void*>(a[6]), reinterpret_cast<const float*>(a[7]),
      reinterpret_cast<const float*>(a[8]), a[9], a[10], a[11],
      reinterpret_cast<const int32_t*>(a[12]), a[13], a[14], reinterpret_cast<const int32_t*>(a[15]),
      reinterpret_cast<const int32_t*>(a[16]), a[17], a[18], a[19], a[20], a[21], a[22],
      (int32_t)a[23], (float)softmax_scale, reinterpret_cast<void*>(a[25]), a[26],
      reinterpret_cast<void*>(a[27]));
}
