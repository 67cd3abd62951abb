// Integer address kernels feeding the append and attention kernels, plus the
// library's error/version plumbing.
//
// Reference behaviour:
//   expand_kv_addresses  kernels/metadata.py:7-24
//   routing_metadata     kernels/routing.py:14-48 (metadata_kernel)
//   routing_slots        kernels/routing.py:7-11 (slots_kernel)
// vrh_sequence_metadata builds a packed step's tables and addresses from lengths that
// live on the GPU (no counterpart in the reference, whose builder is on the host).
#include <stdarg.h>
#include <stdio.h>

#include "common.h"

static thread_local char g_last_error[512] = "";

void vrh_set_error(const char* fmt, ...) {
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(g_last_error, sizeof(g_last_error), fmt, ap);
  va_end(ap);
}

extern "C" const char* vrh_last_error(void) { return g_last_error; }
extern "C" int vrh_abi_version(void) { return 5; }

namespace vrh {
namespace {

__global__ __launch_bounds__(256) void expand_addresses_kernel(
    const int64_t* positions, const int32_t* sequences, const int32_t* tables, int64_t* blocks,
    int64_t* offsets, int64_t n, int32_t width, int32_t page) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= n) return;
  const int64_t pos = positions[i];
  const int64_t seq = sequences[i];
  blocks[i] = tables[seq * width + pos / page];
  offsets[i] = pos % page;
}

// One workgroup per row: lanes copy the row's table slice while lane 0 writes
// the scalars.
__global__ __launch_bounds__(256) void routing_metadata_kernel(
    const int64_t* desc, const int32_t* tables, int64_t* slots, int64_t* positions,
    int32_t* lengths, int64_t* blocks, int64_t* offsets, int32_t* out_tables, int64_t n,
    int32_t width, int32_t page, int32_t planes, int32_t out_width) {
  const int64_t row = blockIdx.x;
  const bool valid = row < n;
  const int64_t slot = valid ? desc[row * 3 + 0] : 0;
  const int64_t depth = valid ? desc[row * 3 + 1] : 0;
  const int64_t pos = valid ? desc[row * 3 + 2] : 0;
  const int64_t plane = planes > 1 ? depth : 0;
  const int64_t base = (slot * planes + plane) * width;
  if (threadIdx.x == 0) {
    slots[row] = slot;
    positions[row] = pos;
    lengths[row] = valid ? (int32_t)(pos + 1) : 0;
    if (valid) {
      blocks[row] = tables[base + pos / page];
      offsets[row] = pos % page;
    }
  }
  for (int c = threadIdx.x; c < out_width; c += 256) {
    out_tables[row * width + c] = valid ? tables[base + c] : 0;
  }
}

__global__ __launch_bounds__(256) void routing_slots_kernel(const int64_t* desc, int64_t* slots,
                                                            int64_t n, int64_t size) {
  const int64_t r = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (r >= size) return;
  slots[r] = r < n ? desc[r * 3] : 0;
}

// Requests that a workgroup's threads scan at a time (four each).
constexpr int kScan = 1024;

struct SequenceArgs {
  const int32_t* tables;
  const int64_t* rows;
  const int32_t* lengths;
  const int32_t* counts;
  int64_t* positions;
  int64_t* blocks;
  int64_t* offsets;
  uint8_t* mask;
  int32_t* out_tables;
  int32_t* out_lengths;
  int32_t* cu;
  int64_t num_rows, table_stride, out_stride, n, tokens;
  int32_t width, out_width, page;
};

// Request r as the step takes it: `length` tokens of which the last `count` are new,
// cut to what the tables hold.
__device__ __forceinline__ void sequence_request(const SequenceArgs& a, int64_t r, int64_t& length,
                                                 int64_t& count) {
  length = max(0, a.lengths[r]);
  count = min((int64_t)max(0, a.counts[r]), length);
  const int64_t row = a.rows[r];
  if (row < 0 || row >= a.num_rows) length = count = 0;
  const int64_t fits = min(length, (int64_t)min(a.width, a.out_width) * a.page);
  count = max((int64_t)0, count - (length - fits));
  length = fits;
}

// Workgroups [0, n): one request each (its table row, length and cumulative count);
// the others 256 tokens each. Every workgroup scans the counts itself, 1024 requests
// at a time: a scan of its own launch would cost more than reading 12 bytes a request
// from L2 again. Bound by latency (two dependent misses and the scan): 64 requests of
// 8000 tokens 4.6 us, 500 requests under tables of 2048 pages (6 MB) 5.7 us.
__global__ __launch_bounds__(256) void sequence_metadata_kernel(SequenceArgs a) {
  __shared__ int64_t ends[kScan];  // where each request's tokens end
  __shared__ int64_t wave_total[4];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const bool request = (int64_t)blockIdx.x < a.n;
  const int64_t t = ((int64_t)blockIdx.x - a.n) * 256 + tid;  // this thread's token
  const int64_t last = request ? (int64_t)blockIdx.x : a.n - 1;  // last request to scan
  int64_t carry = 0;
  int64_t mine = -1, start = 0;  // the token's request, and where its tokens start
  for (int64_t r0 = 0; r0 <= last; r0 += kScan) {
    int64_t sum[4], run = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int64_t r = r0 + tid * 4 + i;
      int64_t length, count = 0;
      if (r <= last) sequence_request(a, r, length, count);
      sum[i] = run += count;
    }
    int64_t before = run;  // inclusive scan over the wave's threads
    for (int m = 1; m < 64; m <<= 1) {
      const int64_t o = __shfl_up(before, m);
      if (lane >= m) before += o;
    }
    __syncthreads();  // the former chunk's ends and totals have been read
    if (lane == 63) wave_total[wave] = before;
    __syncthreads();
    int64_t base = carry + before - run;
    for (int w = 0; w < wave; ++w) base += wave_total[w];
#pragma unroll
    for (int i = 0; i < 4; ++i) ends[tid * 4 + i] = base + sum[i];
    for (int w = 0; w < 4; ++w) carry += wave_total[w];
    __syncthreads();
    if (!request && mine < 0 && t < carry && t < a.tokens) {
      // First request whose tokens end past t.
      int lo = 0, hi = kScan - 1;
      while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (ends[mid] > t) hi = mid; else lo = mid + 1;
      }
      mine = r0 + lo;
      int64_t length, count;
      sequence_request(a, mine, length, count);
      start = ends[lo] - count;
    }
  }
  if (request) {
    const int64_t r = blockIdx.x;
    int64_t length, count;
    sequence_request(a, r, length, count);
    const int64_t end = ends[r % kScan];
    // Tokens past a.tokens have no room: the request's context ends where they do.
    const int64_t cut = min(count, max((int64_t)0, end - a.tokens));
    length -= cut;
    if (tid == 0) {
      a.out_lengths[r] = (int32_t)length;
      a.cu[r + 1] = (int32_t)min(end, a.tokens);
      if (r == 0) a.cu[0] = 0;
    }
    const int used = (int)((length + a.page - 1) / a.page);
    const int32_t* src = a.tables + (used > 0 ? a.rows[r] : 0) * a.table_stride;
    int32_t* dst = a.out_tables + r * a.out_stride;
    for (int c = tid; c < a.out_width; c += 256) dst[c] = c < used ? src[c] : -1;
    return;
  }
  if (a.n == 0 && t == 0) a.cu[0] = 0;
  if (t >= a.tokens) return;
  int64_t position = 0, block = 0;
  if (mine >= 0) {
    int64_t length, count;
    sequence_request(a, mine, length, count);
    position = length - count + (t - start);
    block = a.tables[a.rows[mine] * a.table_stride + position / a.page];
  }
  a.positions[t] = position;
  a.blocks[t] = block;
  a.offsets[t] = position % a.page;
  a.mask[t] = mine >= 0;
}

}  // namespace
}  // namespace vrh

using namespace vrh;

extern "C" int vrh_expand_kv_addresses(const int64_t* positions, const int32_t* sequences,
                                       const int32_t* tables, int64_t* blocks, int64_t* offsets,
                                       int64_t n, int32_t width, int32_t page,
                                       vrh_stream_t stream) {
  VRH_CHECK_ARG(n >= 0 && width >= 0 && page >= 1, "vrh_expand_kv_addresses: bad sizes");
  if (n == 0) return VRH_OK;
  VRH_CHECK_ARG(positions && sequences && tables && blocks && offsets,
                "vrh_expand_kv_addresses: null pointer");
  hipLaunchKernelGGL(expand_addresses_kernel, dim3((unsigned)ceil_div64(n, 256)), dim3(256), 0,
                     (hipStream_t)stream, positions, sequences, tables, blocks, offsets, n, width,
                     page);
  VRH_RETURN_LAUNCH("vrh_expand_kv_addresses");
}

extern "C" int vrh_routing_metadata(const int64_t* descriptors, const int32_t* tables,
                                    int64_t* slots, int64_t* positions, int32_t* lengths,
                                    int64_t* blocks, int64_t* offsets, int32_t* out_tables,
                                    int64_t n, int64_t size, int32_t width, int32_t page,
                                    int32_t planes, int32_t out_width, vrh_stream_t stream) {
  VRH_CHECK_ARG(n >= 0 && size >= n && width >= 1 && page >= 1 && planes >= 1 &&
                    out_width >= 0 && out_width <= width,
                "vrh_routing_metadata: bad sizes n=%lld size=%lld width=%d out_width=%d",
                (long long)n, (long long)size, width, out_width);
  if (size == 0) return VRH_OK;
  VRH_CHECK_ARG(size < (1ll << 31), "vrh_routing_metadata: too many rows");
  VRH_CHECK_ARG(tables && slots && positions && lengths && blocks && offsets && out_tables &&
                    (n == 0 || descriptors),
                "vrh_routing_metadata: null pointer");
  hipLaunchKernelGGL(routing_metadata_kernel, dim3((unsigned)size), dim3(256), 0,
                     (hipStream_t)stream, descriptors, tables, slots, positions, lengths, blocks,
                     offsets, out_tables, n, width, page, planes, out_width);
  VRH_RETURN_LAUNCH("vrh_routing_metadata");
}

extern "C" int vrh_routing_slots(const int64_t* descriptors, int64_t* slots, int64_t n,
                                 int64_t size, vrh_stream_t stream) {
  VRH_CHECK_ARG(n >= 0 && size >= 0, "vrh_routing_slots: bad sizes");
  if (size == 0) return VRH_OK;
  VRH_CHECK_ARG(slots && (n == 0 || descriptors), "vrh_routing_slots: null pointer");
  hipLaunchKernelGGL(routing_slots_kernel, dim3((unsigned)ceil_div64(size, 256)), dim3(256), 0,
                     (hipStream_t)stream, descriptors, slots, n, size);
  VRH_RETURN_LAUNCH("vrh_routing_slots");
}

extern "C" int vrh_sequence_metadata(const int32_t* tables, int64_t num_rows, int64_t table_stride,
                                     const int64_t* table_rows, const int32_t* context_lengths,
                                     const int32_t* query_lengths, int64_t* positions,
                                     int64_t* write_blocks, int64_t* write_offsets,
                                     uint8_t* write_mask, int32_t* out_tables,
                                     int64_t out_table_stride, int32_t* out_lengths,
                                     int32_t* cu_seqlens_q, int64_t n, int64_t tokens, int32_t width,
                                     int32_t out_width, int32_t page, vrh_stream_t stream) {
  static const char* who = "vrh_sequence_metadata";
  VRH_CHECK_ARG(n >= 0 && tokens >= 0 && tokens < (1ll << 31) && num_rows >= 0 && width >= 0 &&
                    out_width >= 0 && page >= 1,
                "%s: bad sizes", who);
  VRH_CHECK_ARG(n + ceil_div64(tokens, 256) < (1ll << 31), "%s: too many requests", who);
  VRH_CHECK_ARG(cu_seqlens_q, "%s: null pointer", who);
  VRH_CHECK_ARG(tokens == 0 || (positions && write_blocks && write_offsets && write_mask),
                "%s: null pointer", who);
  VRH_CHECK_ARG(n == 0 || (table_rows && context_lengths && query_lengths && out_lengths &&
                           (out_tables || out_width == 0) && (tables || num_rows == 0 || width == 0)),
                "%s: null pointer", who);
  VRH_CHECK_ARG(n <= 1 || out_width == 0 || out_table_stride >= out_width, "%s: table rows overlap", who);
  SequenceArgs a;
  a.tables = tables;
  a.rows = table_rows;
  a.lengths = context_lengths;
  a.counts = query_lengths;
  a.positions = positions;
  a.blocks = write_blocks;
  a.offsets = write_offsets;
  a.mask = write_mask;
  a.out_tables = out_tables;
  a.out_lengths = out_lengths;
  a.cu = cu_seqlens_q;
  a.num_rows = num_rows;
  a.table_stride = table_stride;
  a.out_stride = out_table_stride;
  a.n = n;
  a.tokens = tokens;
  a.width = width;
  a.out_width = out_width;
  a.page = page;
  // At least one workgroup, which writes cu[0].
  const int64_t groups = n + ceil_div64(tokens > 0 ? tokens : n == 0, 256);
  hipLaunchKernelGGL(sequence_metadata_kernel, dim3((unsigned)groups), dim3(256), 0,
                     (hipStream_t)stream, a);
  VRH_RETURN_LAUNCH(who);
}
