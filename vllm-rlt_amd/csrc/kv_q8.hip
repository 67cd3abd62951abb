// Writing and reading pages of the 8-bit cache (format: q8.h).
//
// Append. Sequence s holds n = context_lengths[s] tokens after the call, its last
// q = cu[s + 1] - cu[s] (1 without cu) new: rows cu[s] .. of k and v, at positions
// n - q .. n - 1 of its block table. For every page with a new position, every KV
// head, and K and V apart, with a = max |x| over the page's new finite values:
//   e' = least exponent with a <= 448 * 2^(e' - 127)
//   e  = the page holds older tokens of the sequence ? max(e', its exponent) : e'
//   new byte = e4m3(x * 2^(127 - e)), older byte = e4m3(old * 2^(e_old - e))
// The sequence form (not one address per row) is what tells a page's older tokens
// from bytes that a former owner left, without any state beside the scales.
//
// One wave per (page, head, K or V): it alone reads and writes that scale and those
// bytes, so there are no atomics and no order to depend on. Bound by HBM: a row is
// read once (its values stay in registers between the maximum and the rounding) and
// half of it written. 8000 rows in 16 chunks and 39 single rows (16 x 128, bf16): 26 us, as
// their pages take to be read back, 4.0 TB/s where a large copy reaches 4.75. A decode
// step's 64 rows: 5.6 us, three dependent misses (length, page id, scale).
#include "q8.h"

namespace vrh {
namespace {

struct Q8AppendArgs {
  uint8_t* k_cache;
  uint8_t* v_cache;
  uint8_t* scales;
  const void* k;
  const void* v;
  const int32_t* tables;
  const int32_t* lengths;
  const int32_t* cu;  // null: one row per sequence
  int64_t c_block, c_token, c_head;
  int64_t s_block, s_head;
  int64_t k_row, k_head, v_row, v_head;
  int64_t num_seqs, total_q, num_blocks, table_stride, slot_base;
  int32_t heads, head_dim, block_size, table_width;
  int32_t shift;  // log2(vectors per head) or -1
};

// A wave's page: the first page slots of sequence s are floor(cu[s] / bs) + 2 s, which
// leaves it at least as many as its q tokens can touch (floor(q / bs) + 2), so that a
// slot finds its sequence without a prefix sum of pages. 64 candidates at a time; what
// is needed of the last 64 sequences is loaded with them, so that up to 64 sequences
// cost one round trip to memory.
struct Q8Slot {
  int64_t seq, row0, q, n;  // the sequence, its first row, rows and length
  int page_idx;
};
__device__ __forceinline__ int64_t pick64(int64_t x, int lane) {
  return ((int64_t)__builtin_amdgcn_readlane((int)(x >> 32), lane) << 32) |
         (uint32_t)__builtin_amdgcn_readlane((int)x, lane);
}
__device__ __forceinline__ bool q8_slot(const Q8AppendArgs& a, int64_t slot, Q8Slot& s) {
  const int lane = threadIdx.x & 63;
  if (a.cu == nullptr) {
    if (slot >= a.num_seqs) return false;
    s = {slot, slot, 1, a.lengths[slot], 0};
    return true;
  }
  int64_t lo = 0, hi = a.num_seqs;  // the sequence is in [lo, hi)
  for (;;) {
    const int64_t step = (hi - lo + 63) / 64;
    const int64_t mine = lo + lane * step;
    int64_t first = 0;
    int q = 0, n = 0;
    if (mine < hi) {
      first = a.cu[mine];
      if (step == 1) {
        q = a.cu[mine + 1] - (int)first;
        n = a.lengths[mine];
      }
    }
    const uint64_t hit = __ballot(mine < hi && first / a.block_size + 2 * mine <= slot);
    if (hit == 0) return false;
    const int pick = 63 - __builtin_clzll(hit);
    lo += pick * step;
    if (step == 1) {
      s.seq = lo;
      s.row0 = pick64(first, pick);
      s.q = __builtin_amdgcn_readlane(q, pick);
      s.n = __builtin_amdgcn_readlane(n, pick);
      s.page_idx = (int)(slot - (s.row0 / a.block_size + 2 * lo));
      return true;
    }
    hi = min(hi, lo + step);
  }
}

template <typename T, int VE>
struct Q8Vec {
  using raw_t = raw_of<VE * (int)sizeof(T)>;
  using q_t = raw_of<VE>;
};

template <int VE>
__device__ __forceinline__ void q8_store(uint8_t* p, const float (&x)[VE], float inv) {
  if constexpr (VE == 1) {
    *p = q8_from_f32(x[0] * inv);
  } else {
    union {
      raw_of<VE> raw;
      uint32_t w[VE / 4];
    } u;
#pragma unroll
    for (int i = 0; i < VE; i += 4) u.w[i / 4] = q8_pack4(x[i] * inv, x[i + 1] * inv, x[i + 2] * inv, x[i + 3] * inv);
    *reinterpret_cast<raw_of<VE>*>(p) = u.raw;
  }
}

template <int VE>
__device__ __forceinline__ void q8_load(const uint8_t* p, float (&x)[VE]) {
  if constexpr (VE == 1) {
    x[0] = q8_to_f32(*p);
  } else {
    union {
      raw_of<VE> raw;
      uint32_t w[VE / 4];
    } u;
    u.raw = *reinterpret_cast<const raw_of<VE>*>(p);
#pragma unroll
    for (int i = 0; i < VE; i += 4) {
      float f[4];
      q8_unpack4(u.w[i / 4], f);
#pragma unroll
      for (int j = 0; j < 4; ++j) x[i + j] = f[j];
    }
  }
}

constexpr int kHeld = 4;  // vectors a lane keeps between the two passes

template <typename T, int VE>
__global__ __launch_bounds__(256) void kv_append_q8_kernel(Q8AppendArgs a) {
  using raw_t = typename Q8Vec<T, VE>::raw_t;
  const int lane = threadIdx.x & 63;
  const int item = (int)__builtin_amdgcn_readfirstlane(blockIdx.y * 4 + (threadIdx.x >> 6));
  if (item >= 2 * a.heads) return;
  const int head = item >> 1, part = item & 1;
  Q8Slot at;
  if (!q8_slot(a, a.slot_base + blockIdx.x, at)) return;
  const int64_t row0 = at.row0, q = at.q, n = at.n;
  if (q <= 0 || n <= 0) return;
  // Positions before 0 or past the table take no row.
  const int64_t before = n - q;  // may be negative: then the first rows have no position
  const int64_t first = before > 0 ? before : 0;
  const int64_t cap = (int64_t)a.table_width * a.block_size;
  const int64_t end = n < cap ? n : cap;
  const int64_t page = first / a.block_size + at.page_idx;
  const int64_t p0 = page * a.block_size;
  if (p0 >= end) return;
  const int64_t block = a.tables[at.seq * a.table_stride + page];
  if (block < 0 || block >= a.num_blocks) return;
  const int old = (int)max((int64_t)0, first - p0);  // older tokens of the page
  const int stop = (int)min((int64_t)a.block_size, end - p0);
  int64_t row = row0 + (p0 + old - before);  // row of the page's first new token
  int count = stop - old;
  if (row < 0 || row >= a.total_q) return;
  count = (int)min((int64_t)count, a.total_q - row);

  const T* src = reinterpret_cast<const T*>(part ? a.v : a.k) + (int64_t)head * (part ? a.v_head : a.k_head);
  const int64_t src_row = part ? a.v_row : a.k_row;
  uint8_t* dst = (part ? a.v_cache : a.k_cache) + block * a.c_block + head * a.c_head;
  uint8_t* scale = a.scales + block * a.s_block + head * a.s_head + part;
  const int per_token = a.head_dim / VE;
  const int vecs = count * per_token;
  auto split = [&](int i, int& token, int& v) {
    if (a.shift >= 0) {
      token = i >> a.shift;
      v = i & (per_token - 1);
    } else {
      token = i / per_token;
      v = i - token * per_token;
    }
  };
  auto load = [&](int i) {
    int token, v;
    split(i, token, v);
    return *reinterpret_cast<const raw_t*>(src + (row + token) * src_row + v * VE);
  };
  auto values = [&](raw_t r, float (&x)[VE]) { unpack<T, VE>(r, x); };
  raw_t held[kHeld];
#pragma unroll
  for (int u = 0; u < kHeld; ++u)
    if (u * 64 + lane < vecs) held[u] = load(u * 64 + lane);
  const int e_old = old > 0 ? *scale : 0;
  float amax = 0.f;
  auto take = [&](raw_t r) {
    float x[VE];
    values(r, x);
#pragma unroll
    for (int i = 0; i < VE; ++i) {
      const float m = fabsf(x[i]);
      amax = fmaxf(amax, m < INFINITY ? m : 0.f);
    }
  };
#pragma unroll
  for (int u = 0; u < kHeld; ++u)
    if (u * 64 + lane < vecs) take(held[u]);
  for (int i = kHeld * 64 + lane; i < vecs; i += 64) take(load(i));
  amax = wave_max(amax);
  const int e = max(q8_exponent(amax), e_old);
  const float inv = q8_scale(254 - e);
  auto put = [&](int i, raw_t r) {
    int token, v;
    split(i, token, v);
    float x[VE];
    values(r, x);
    q8_store<VE>(dst + (int64_t)(old + token) * a.c_token + v * VE, x, inv);
  };
#pragma unroll
  for (int u = 0; u < kHeld; ++u)
    if (u * 64 + lane < vecs) put(u * 64 + lane, held[u]);
  for (int i = kHeld * 64 + lane; i < vecs; i += 64) put(i, load(i));
  if (old > 0 && e > e_old) {
    const float f = q8_scale(max(0, 127 + e_old - e));
    for (int i = lane; i < old * per_token; i += 64) {
      int token, v;
      split(i, token, v);
      uint8_t* p = dst + (int64_t)token * a.c_token + v * VE;
      float x[VE];
      q8_load<VE>(p, x);
      q8_store<VE>(p, x, f);
    }
  }
  if (lane == 0) *scale = (uint8_t)e;
}

struct Q8ReadArgs {
  void* out_k;
  void* out_v;
  const uint8_t* k_cache;
  const uint8_t* v_cache;
  const uint8_t* scales;
  const int64_t* pages;
  int64_t c_block, c_token, c_head;
  int64_t s_block, s_head;
  int64_t num_blocks, page_base;
  int32_t heads, head_dim, block_size;
};

// One wave per (listed page, head, K or V); a page outside the pool reads as zeros.
template <typename T, int VE>
__global__ __launch_bounds__(256) void kv_read_q8_kernel(Q8ReadArgs a) {
  const int lane = threadIdx.x & 63;
  const int item = (int)__builtin_amdgcn_readfirstlane(blockIdx.y * 4 + (threadIdx.x >> 6));
  if (item >= 2 * a.heads) return;
  const int head = item >> 1, part = item & 1;
  const int64_t i = a.page_base + blockIdx.x;
  const int64_t block = a.pages[i];
  const bool ok = block >= 0 && block < a.num_blocks;
  const uint8_t* src = (part ? a.v_cache : a.k_cache) + (ok ? block : 0) * a.c_block + head * a.c_head;
  const float scale = ok ? q8_scale(a.scales[block * a.s_block + head * a.s_head + part]) : 0.f;
  T* dst = reinterpret_cast<T*>(part ? a.out_v : a.out_k) + (i * a.block_size * a.heads + head) * a.head_dim;
  const int per_token = a.head_dim / VE;
  for (int j = lane; j < a.block_size * per_token; j += 64) {
    const int token = j / per_token, v = j - token * per_token;
    float x[VE] = {};
    if (ok) q8_load<VE>(src + (int64_t)token * a.c_token + v * VE, x);
#pragma unroll
    for (int c = 0; c < VE; ++c) x[c] *= scale;
    T* p = dst + (int64_t)token * a.heads * a.head_dim + v * VE;
    if constexpr (VE * (int)sizeof(T) <= 16) {
      store_raw<T, VE>(p, pack<T, VE>(x));
    } else {
      constexpr int H = 16 / (int)sizeof(T);
#pragma unroll
      for (int c = 0; c < VE; c += H) {
        float y[H];
#pragma unroll
        for (int d = 0; d < H; ++d) y[d] = x[c + d];
        store_raw<T, H>(p + c, pack<T, H>(y));
      }
    }
  }
}

constexpr int64_t kMostPages = 1ll << 23;  // per launch: of 256 threads each, less than 2^32

// Whether vectors of `ve` elements keep every access of a kernel aligned.
bool aligned_vectors(int ve, int es, int64_t head_dim, std::initializer_list<int64_t> cache_strides,
                     std::initializer_list<int64_t> row_strides, std::initializer_list<const void*> caches,
                     std::initializer_list<const void*> rows) {
  if (head_dim % ve) return false;
  for (int64_t s : cache_strides)
    if (s % ve) return false;
  for (int64_t s : row_strides)
    if (s % ve) return false;
  for (const void* p : caches)
    if ((uintptr_t)p % ve) return false;
  for (const void* p : rows)
    if ((uintptr_t)p % ((size_t)ve * es > 16 ? 16 : ve * es)) return false;
  return true;
}

}  // namespace
}  // namespace vrh

using namespace vrh;

extern "C" int vrh_kv_append_q8(int dtype, void* key_cache, void* value_cache, void* scales,
                                int64_t cache_block_stride, int64_t cache_token_stride,
                                int64_t cache_head_stride, int64_t scale_block_stride,
                                int64_t scale_head_stride, const void* k, const void* v,
                                int64_t k_row_stride, int64_t k_head_stride, int64_t v_row_stride,
                                int64_t v_head_stride, const int32_t* block_tables,
                                const int32_t* context_lengths, const int32_t* cu_seqlens_q,
                                int64_t num_seqs, int64_t total_q, int32_t kv_heads,
                                int32_t head_dim, int64_t num_blocks, int32_t block_size,
                                int32_t table_width, int64_t table_stride, vrh_stream_t stream) {
  static const char* who = "vrh_kv_append_q8";
  const int es = dtype_bytes(dtype);
  VRH_CHECK_ARG(es > 0, "%s: unknown dtype %d", who, dtype);
  VRH_CHECK_ARG(num_seqs >= 0 && total_q >= 0 && kv_heads >= 1 && head_dim >= 1 && num_blocks >= 0 &&
                    block_size >= 1 && table_width >= 0,
                "%s: bad sizes", who);
  VRH_CHECK_ARG(kv_heads <= 32767 * 4 && (int64_t)block_size * head_dim < (1ll << 30),
                "%s: page too large", who);
  VRH_CHECK_ARG(cu_seqlens_q || total_q == num_seqs,
                "%s: without cu_seqlens_q there is one row per sequence", who);
  if (num_seqs == 0 || total_q == 0 || table_width == 0 || num_blocks == 0) return VRH_OK;
  VRH_CHECK_ARG(key_cache && value_cache && scales && k && v && block_tables && context_lengths,
                "%s: null pointer", who);
  const int64_t slots = cu_seqlens_q ? total_q / block_size + 2 * num_seqs : num_seqs;
  Q8AppendArgs a;
  a.k_cache = (uint8_t*)key_cache;
  a.v_cache = (uint8_t*)value_cache;
  a.scales = (uint8_t*)scales;
  a.k = k;
  a.v = v;
  a.tables = block_tables;
  a.lengths = context_lengths;
  a.cu = cu_seqlens_q;
  a.c_block = cache_block_stride;
  a.c_token = cache_token_stride;
  a.c_head = cache_head_stride;
  a.s_block = scale_block_stride;
  a.s_head = scale_head_stride;
  a.k_row = k_row_stride;
  a.k_head = k_head_stride;
  a.v_row = v_row_stride;
  a.v_head = v_head_stride;
  a.num_seqs = num_seqs;
  a.total_q = total_q;
  a.num_blocks = num_blocks;
  a.table_stride = table_stride;
  a.heads = kv_heads;
  a.head_dim = head_dim;
  a.block_size = block_size;
  a.table_width = table_width;
  const int ve = 16 / es;
  const bool wide = aligned_vectors(
      ve, es, head_dim, {cache_block_stride, cache_token_stride, cache_head_stride},
      {k_row_stride, k_head_stride, v_row_stride, v_head_stride}, {key_cache, value_cache}, {k, v});
  const int per_token = wide ? head_dim / ve : head_dim;
  a.shift = (per_token & (per_token - 1)) == 0 ? __builtin_ctz((unsigned)per_token) : -1;
  hipStream_t s = (hipStream_t)stream;
  for (int64_t first = 0; first < slots; first += kMostPages) {
    a.slot_base = first;
    const dim3 grid((unsigned)(slots - first < kMostPages ? slots - first : kMostPages),
                    (unsigned)ceil_div(2 * kv_heads, 4));
#define VRH_APPEND(T)                                                                                 \
  if (wide) hipLaunchKernelGGL((kv_append_q8_kernel<T, 16 / sizeof(T)>), grid, dim3(256), 0, s, a); \
  else hipLaunchKernelGGL((kv_append_q8_kernel<T, 1>), grid, dim3(256), 0, s, a);
    if (dtype == VRH_DTYPE_F32) {
      VRH_APPEND(float)
    } else if (dtype == VRH_DTYPE_F16) {
      VRH_APPEND(f16_t)
    } else {
      VRH_APPEND(bf16_t)
    }
#undef VRH_APPEND
  }
  VRH_RETURN_LAUNCH(who);
}

extern "C" int vrh_kv_read_q8(int dtype, void* out_k, void* out_v, const void* key_cache,
                              const void* value_cache, const void* scales,
                              int64_t cache_block_stride, int64_t cache_token_stride,
                              int64_t cache_head_stride, int64_t scale_block_stride,
                              int64_t scale_head_stride, const int64_t* pages, int64_t num_pages,
                              int32_t kv_heads, int32_t head_dim, int64_t num_blocks,
                              int32_t block_size, vrh_stream_t stream) {
  static const char* who = "vrh_kv_read_q8";
  const int es = dtype_bytes(dtype);
  VRH_CHECK_ARG(es > 0, "%s: unknown dtype %d", who, dtype);
  VRH_CHECK_ARG(num_pages >= 0 && kv_heads >= 1 && head_dim >= 1 && num_blocks >= 0 && block_size >= 1,
                "%s: bad sizes", who);
  VRH_CHECK_ARG(kv_heads <= 32767 * 4 && (int64_t)block_size * head_dim < (1ll << 30),
                "%s: page too large", who);
  if (num_pages == 0) return VRH_OK;
  VRH_CHECK_ARG(out_k && out_v && key_cache && value_cache && scales && pages, "%s: null pointer", who);
  Q8ReadArgs a;
  a.out_k = out_k;
  a.out_v = out_v;
  a.k_cache = (const uint8_t*)key_cache;
  a.v_cache = (const uint8_t*)value_cache;
  a.scales = (const uint8_t*)scales;
  a.pages = pages;
  a.c_block = cache_block_stride;
  a.c_token = cache_token_stride;
  a.c_head = cache_head_stride;
  a.s_block = scale_block_stride;
  a.s_head = scale_head_stride;
  a.num_blocks = num_blocks;
  a.heads = kv_heads;
  a.head_dim = head_dim;
  a.block_size = block_size;
  const bool wide = aligned_vectors(16, es, head_dim,
                                    {cache_block_stride, cache_token_stride, cache_head_stride}, {},
                                    {key_cache, value_cache}, {out_k, out_v});
  hipStream_t s = (hipStream_t)stream;
  for (int64_t first = 0; first < num_pages; first += kMostPages) {
    a.page_base = first;
    const dim3 grid((unsigned)(num_pages - first < kMostPages ? num_pages - first : kMostPages),
                    (unsigned)ceil_div(2 * kv_heads, 4));
#define VRH_READ(T)                                                                     \
  if (wide) hipLaunchKernelGGL((kv_read_q8_kernel<T, 16>), grid, dim3(256), 0, s, a);   \
  else hipLaunchKernelGGL((kv_read_q8_kernel<T, 1>), grid, dim3(256), 0, s, a);
    if (dtype == VRH_DTYPE_F32) {
      VRH_READ(float)
    } else if (dtype == VRH_DTYPE_F16) {
      VRH_READ(f16_t)
    } else {
      VRH_READ(bf16_t)
    }
#undef VRH_READ
  }
  VRH_RETURN_LAUNCH(who);
}
