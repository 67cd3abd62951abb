// Paged single-query (decode) attention over the 8-bit cache (format: q8.h).
//
// out[r, h] = softmax_t(q[r, h] . K_t / sqrt(D)) V_t over the visible tokens t of row
// r, K_t = e4m3 * 2^(ek - 127) of t's page and KV head h / group, V_t likewise.
//
// One pass over the keys with the running maximum and sum of the softmax; a row's
// keys are cut into splits of whole pages whose (max, sum, accumulator) are merged
// in split order. The cut depends on the row's own length only, so a row's result
// does not depend on the batch, and a packed query equals a decode row bit for bit.
//
// Bound by HBM: 2 bytes per visible token, KV head and dim. 64 rows of 512-4096 tokens
// (16 x 128 heads, bf16, 607 MB): 107 us, 5.7 TB/s, and 5 us of merge. Lone rows and short
// ones are bound by latency: length, page ids, K and V, merge.
#include <algorithm>
#include <type_traits>

#include "decode_q8.h"

namespace vrh {
namespace {

__device__ __forceinline__ int page_of(int pos, const DecodeQ8Args& a) {
  return a.d.bs_shift >= 0 ? pos >> a.d.bs_shift : pos / a.d.block_size;
}

// Sum over the lanes up to this one.
__device__ __forceinline__ int wave_scan(int x) {
  x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xF, 0xF, true);  // row_shr:1
  x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xF, 0xF, true);
  x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xF, 0xF, true);
  x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xF, 0xF, true);
  x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xA, 0xF, false);  // row_bcast:15
  x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xC, 0xF, false);  // row_bcast:31
  return x;
}

// Work of the waves. For up to kCompactRows rows the splits that exist are numbered (rows
// in order), each wave counting them itself, 64 rows at a time, and as many waves as are
// resident take every waves-th one: none is launched without work however wide the
// tables are (38 float32 rows of 2-21 tokens, 64 heads, under tables of 2063 pages: 137 us
// with a wave for each slot), and the waves of a split's heads, whose pages are
// neighbours in memory, run at the same time. Which wave takes a split changes no
// result. Equal shares of consecutive splits, with no restart between them, were slower
// (64 rows of 512-4096 tokens, 16 x 128 heads: 117 us against 107): the heads drift apart.
// Beyond that many rows a wave takes one split, workgroups being dealt slots x rows.
constexpr int kCompactRows = 512;
constexpr int kSegment = 64;

// A lane's row of up to 64 consecutive ones, and its splits.
struct RowQ8 {
  int64_t trow, qrow;
  int n, splits;
};
__device__ __forceinline__ RowQ8 q8_row(const DecodeQ8Args& a, int64_t row) {
  RowQ8 r = {0, 0, -1, 0};
  if (row < a.d.rows) r.n = row_length(row, a.d, &r.trow, &r.qrow);
  if (r.n > 0) r.splits = partition_q8(r.n, a).nsplit;
  else if (r.n == 0) r.splits = 1;
  return r;
}

struct ItemQ8 {
  int64_t row;   // work row
  int64_t trow;  // table row
  int64_t qrow;  // query and output row
  int n;         // visible length
  int split;
};

// A wave's walk over the splits, all of it wave-uniform but `r` and `upto`.
struct WalkQ8 {
  RowQ8 r;          // this lane's row of the 64 from `base` on
  int upto;         // splits of those rows up to this lane's
  int64_t base;
  uint32_t before;  // splits of the rows before `base`
  uint32_t next;
};

__device__ __forceinline__ void q8_start(const DecodeQ8Args& a, uint32_t wave, WalkQ8& w) {
  w.next = wave;
  if (a.compact == 0) return;
  w.base = 0;
  w.before = 0;
  w.r = q8_row(a, threadIdx.x & 63);
  w.upto = wave_scan(w.r.splits);
}

// The walk's next split; false when there is none. `step`: waves that walk together.
__device__ __forceinline__ bool q8_next(const DecodeQ8Args& a, uint32_t step, WalkQ8& w, ItemQ8& it) {
  if (a.compact == 0) {
    if (w.next == UINT32_MAX) return false;
    it.row = a.d.row_base + w.next / (uint32_t)a.slots;
    it.split = (int)(w.next % (uint32_t)a.slots);
    it.n = row_length(it.row, a.d, &it.trow, &it.qrow);
    w.next = UINT32_MAX;
    return true;
  }
  for (;;) {
    const uint32_t all = (uint32_t)__builtin_amdgcn_readlane(w.upto, 63);
    if (w.next - w.before < all) break;
    w.before += all;
    w.base += 64;
    if (w.base >= a.d.rows) return false;
    w.r = q8_row(a, w.base + (threadIdx.x & 63));
    w.upto = wave_scan(w.r.splits);
  }
  // First lane whose splits end past the next one.
  const uint32_t at = w.next - w.before;
  const int pick = __builtin_ffsll((long long)__ballot((uint32_t)w.upto > at)) - 1;
  it.row = w.base + pick;
  it.trow = ((int64_t)__builtin_amdgcn_readlane((int)(w.r.trow >> 32), pick) << 32) |
            (uint32_t)__builtin_amdgcn_readlane((int)w.r.trow, pick);
  it.qrow = ((int64_t)__builtin_amdgcn_readlane((int)(w.r.qrow >> 32), pick) << 32) |
            (uint32_t)__builtin_amdgcn_readlane((int)w.r.qrow, pick);
  it.n = __builtin_amdgcn_readlane(w.r.n, pick);
  it.split = (int)at - (__builtin_amdgcn_readlane(w.upto, pick) - __builtin_amdgcn_readlane(w.r.splits, pick));
  w.next += step;
  return true;
}

// ------------------------------------------------------ any shape, VALU
// One wave per (split, q head, row). LPT lanes cover a token's head_dim with VE
// elements each (ND vectors of VE, LPT * VE apart, where that is not enough), so a
// wave load covers 64 / LPT tokens; U such loads of K and of V are issued back to
// back. Each token group keeps its own softmax state, merged once per split. All
// arithmetic is fp32. For the shapes that the matrix kernel does not take: other head
// dims, block sizes and alignments. It reads a KV head once per q head (37 rows of
// 300-6000 tokens, 32 over 8 heads, 187 us against 48 of the matrix kernel).
template <typename T, int VE, int LPT, int ND>
__global__ __launch_bounds__(64) void paged_decode_q8_kernel(DecodeQ8Args a) {
  constexpr int U = VE >= 16 ? 8 : VE >= 4 ? 4 : 2;
  constexpr int TPL = 64 / LPT;
  constexpr int CH = U * TPL;
  using raw_t = raw_of<VE>;
  const int lane = threadIdx.x;
  const int dg = lane % LPT, tg = lane / LPT;
  const uint32_t first = blockIdx.x / (uint32_t)a.units, step = gridDim.x / (uint32_t)a.units;
  const int head = (int)(blockIdx.x - first * (uint32_t)a.units);
  const int kvh = head / a.d.group;
  WalkQ8 walk;
  q8_start(a, first, walk);
  ItemQ8 it;
  while (q8_next(a, step, walk, it)) {
    const int n = it.n, split = it.split;
    T* out = reinterpret_cast<T*>(a.d.out) + it.qrow * a.d.o_row + (int64_t)head * a.d.o_head;
    if (n <= 0) {
      if (n == 0 && split == 0)
        for (int d = lane; d < a.d.head_dim; d += 64) out[d] = from_f32<T>(0.f);
      continue;
    }
    const PartitionQ8 P = partition_q8(n, a);
    if (split >= P.nsplit) continue;

    float qf[ND][VE], acc[ND][VE];
    int dim[ND];  // this lane's dims, clamped into the row (their q is zero, they store nothing)
    bool dvalid[ND];
    const T* qp = reinterpret_cast<const T*>(a.d.q) + it.qrow * a.d.q_row + (int64_t)head * a.d.q_head;
#pragma unroll
    for (int j = 0; j < ND; ++j) {
      const int d0 = (j * LPT + dg) * VE;
      dvalid[j] = d0 < a.d.head_dim;
      dim[j] = dvalid[j] ? d0 : 0;
#pragma unroll
      for (int i = 0; i < VE; ++i) {
        qf[j][i] = dvalid[j] ? to_f32(qp[dim[j] + i]) * a.d.scale_log2 : 0.f;
        acc[j][i] = 0.f;
      }
    }
    const uint8_t* kbase = reinterpret_cast<const uint8_t*>(a.d.k) + (int64_t)kvh * a.d.k_head;
    const uint8_t* vbase = reinterpret_cast<const uint8_t*>(a.d.v) + (int64_t)kvh * a.d.v_head;
    const uint8_t* sbase = a.scales + (int64_t)kvh * a.s_head;
    const int32_t* table = a.d.tables + it.trow * a.d.table_stride;
    const int s0 = P.first + split * P.bps, s1 = min(s0 + P.bps, P.first + P.pages);
    float m = -INFINITY, l = 0.f;

    for (int seg = s0; seg < s1; seg += 64) {
      // Up to 64 page ids and their scales, one page a lane.
      const int seg1 = min(s1, seg + 64);
      const int blk = seg + lane < seg1 ? pool_block(table[seg + lane], a) : 0;
      const uint32_t ex = q8_exponents(sbase + (int64_t)blk * a.s_block);
      // (int64: the last page's end may lie past 2^31 tokens)
      const int tb = max(P.start, seg * a.d.block_size);
      const int te = (int)min((int64_t)n, (int64_t)seg1 * a.d.block_size);
      for (int left = te - tb; left > 0; left -= CH) {
        const int p0 = te - left;
        raw_t kr[U][ND], vr[U][ND];
        float ks[U], vs[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          // Positions past the end read the last token again (and are masked).
          const int pos = left > u * TPL + tg ? p0 + u * TPL + tg : te - 1;
          int page, off;
          if (a.d.bs_shift >= 0) {
            page = pos >> a.d.bs_shift;
            off = pos & (a.d.block_size - 1);
          } else {
            page = pos / a.d.block_size;
            off = pos - page * a.d.block_size;
          }
          const int64_t b = shfl_i32(blk, page - seg);
          const uint32_t e = (uint32_t)shfl_i32((int)ex, page - seg);
          ks[u] = q8_scale(e & 255);
          vs[u] = q8_scale(e >> 8);
#pragma unroll
          for (int j = 0; j < ND; ++j) {
            kr[u][j] = __builtin_nontemporal_load(reinterpret_cast<const raw_t*>(
                kbase + b * a.d.k_block + (int64_t)off * a.d.k_token + dim[j]));
            vr[u][j] = __builtin_nontemporal_load(reinterpret_cast<const raw_t*>(
                vbase + b * a.d.v_block + (int64_t)off * a.d.v_token + dim[j]));
          }
        }
        float sc[U], mx = m;
#pragma unroll
        for (int u = 0; u < U; ++u) {
          float d = 0.f;
#pragma unroll
          for (int j = 0; j < ND; ++j) {
            float x[VE];
            q8_values<VE>(kr[u][j], x);
#pragma unroll
            for (int i = 0; i < VE; ++i) d = fmaf(qf[j][i], x[i], d);
          }
          d = group_sum<LPT>(d) * ks[u];
          sc[u] = left > u * TPL + tg ? d : -INFINITY;
          mx = fmaxf(mx, sc[u]);
        }
        const float safe = mx == -INFINITY ? 0.f : mx;
        const float corr = fast_exp2(m - safe);
        l *= corr;
#pragma unroll
        for (int j = 0; j < ND; ++j)
#pragma unroll
          for (int i = 0; i < VE; ++i) acc[j][i] *= corr;
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const float p = fast_exp2(sc[u] - safe);
          l += p;
          const float w = p * vs[u];
          // A masked token's weight is 0, and its value must not matter (0 * NaN).
          const bool seen = left > u * TPL + tg;
#pragma unroll
          for (int j = 0; j < ND; ++j) {
            float x[VE];
            q8_values<VE>(vr[u][j], x);
#pragma unroll
            for (int i = 0; i < VE; ++i) acc[j][i] = seen ? fmaf(w, x[i], acc[j][i]) : acc[j][i];
          }
        }
        m = mx;
      }
    }
    // Merge the token groups' states.
    const float M = cross_group_max<LPT>(m);
    // (l is 0 only where the group saw no token: a NaN score leaves m at -inf too)
    const float w = l == 0.f ? 0.f : fast_exp2(m - M);
    const float L = cross_group_sum<LPT>(l * w);
#pragma unroll
    for (int j = 0; j < ND; ++j)
#pragma unroll
      for (int i = 0; i < VE; ++i) acc[j][i] = cross_group_sum<LPT>(acc[j][i] * w);
    if (tg != 0) continue;
    if (P.nsplit == 1) {
      const float inv = 1.f / L;
#pragma unroll
      for (int j = 0; j < ND; ++j)
#pragma unroll
        for (int i = 0; i < VE; ++i)
          if (dvalid[j]) out[dim[j] + i] = from_f32<T>(acc[j][i] * inv);
      continue;
    }
    const int64_t idx = (it.row * a.d.q_heads + head) * a.slots + split;
    if (dg == 0) {
      a.d.part_ml[idx * 2] = M;
      a.d.part_ml[idx * 2 + 1] = L;
    }
    float* dst = a.d.part_acc + idx * a.d.head_dim;
#pragma unroll
    for (int j = 0; j < ND; ++j)
#pragma unroll
      for (int i = 0; i < VE; ++i)
        if (dvalid[j]) dst[dim[j] + i] = acc[j][i];
  }
}

// ------------------------------------------------------------- on MFMA
// One wave per (split, KV head, row) serves up to 16 q heads of the KV head (the
// columns of v_mfma_f32_16x16x32; groups of more take several waves):
//  * K and V come in chunks of 32 tokens straight into a ring of kStages wave-private
//    LDS stages, kStages - 1 chunks ahead: no registers are held by loads in flight and no
//    barrier is needed. One load instruction covers
//    RPI whole rows; the block size is a power of two of at least 16, so 16-token steps
//    lie in one page and take one (scalar) address.
//  * S^T = K Q^T per 16 tokens: bytes are converted to the query's type (exact), 16 a
//    lane per LDS read, which is two k-steps; the dims of Q^T's k-slots follow that
//    order. The page's K scale joins the softmax scale on the fp32 scores.
//  * O^T += V^T P^T per 32 tokens: the S accumulators, rounded to the query's type, are
//    the P^T operand; one ds_read_b64_tr_b8 returns 8 tokens of a dim for V^T, whose
//    conversion applies the page's scale (exact in bf16; in f16 see v_scale).
//  * float32 queries and weights are three bf16 pieces each (24 bits: nothing is rounded),
//    three MFMAs for one, while K and V are exact in bf16 already: 17 rows of 1500-2600
//    tokens (32 over 8 heads, D = 64) 39 us in the VALU kernel, 16 here; 16 rows of about
//    1900 tokens (16 x 64 heads) 22 and 18.
//  * A row of LDS is D bytes of 16-byte chunks, chunk c of row r stored at slot
//    c ^ swizzle(r), so that both readers spread over all banks.
// A stage is 8 KiB at head_dim 128: two of them leave nine waves to a CU, and it is other
// waves that cover a chunk's chain of LDS reads, MFMAs and exponentials (about 1800
// cycles). Asked for three waves a SIMD the compiler keeps the accumulators out of AGPRs
// and needs 127 registers (165 with float32) instead of 171. Three stages and six waves: 64 rows of 512-4096 tokens
// (16 x 128 heads) 112 us instead of 110, 37 float16 rows of 32 over 8 heads 51 instead of
// 48, 24 rows with a window of 1024 23.6 instead of 20.4. Without the arithmetic those 64
// rows take 101 us (6.0 TB/s), without the loads 75.
constexpr int kChunk = 32;  // tokens per stage
constexpr int kStages = 2;

typedef __attribute__((ext_vector_type(4))) float f32x4_t;
typedef __attribute__((ext_vector_type(4))) uint32_t u32x4_t;
typedef __attribute__((ext_vector_type(2))) uint32_t u32x2_t;

// ds_read_b64_tr_b8: within each 16-lane group lane j receives byte j % 8 of the 8-byte
// chunks addressed by lanes 2i + j / 8, i = 0..7 (byte i of the result): lanes 2i, 2i + 1
// that address 16 bytes of row i give lane j column j of rows 0..7.
__device__ __forceinline__ u32x2_t lds_tr8(uint32_t offset) {
  typedef int v2i __attribute__((ext_vector_type(2)));
  const v2i r = __builtin_amdgcn_ds_read_tr8_b64_v2i32(
      (v2i __attribute__((address_space(3)))*)(uintptr_t)offset);
  return __builtin_bit_cast(u32x2_t, r);
}

template <int D>
__device__ __forceinline__ int q8_swizzle(int row) {
  if constexpr (D == 128) {
    const int i = row >> 1;
    return (i & 3) | (((i >> 2) ^ (i >> 3)) & 1) << 2;
  } else {
    const int i = row >> 2;
    return (i & 1) | (((i >> 1) ^ (i >> 2)) & 1) << 1;
  }
}

// global_load_lds_dword: 4 bytes per lane to m0 + 4 * lane (see lds_dma16).
__device__ __forceinline__ void lds_dma4(const void* g, uint32_t m0) {
  asm volatile("s_nop 0\n\tglobal_load_lds_dword %0, off" ::"v"(g), "{m0}"(m0) : "memory");
}

__device__ __forceinline__ float readlane_f32(float x, int lane) {
  return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(x), lane));
}

// Two floats as three bf16 pairs each that sum to them: sink(piece, pair). A float has 24
// significant bits and a piece takes the next 8, so nothing is rounded.
template <typename Sink>
__device__ __forceinline__ void split3(float a, float b, Sink sink) {
#pragma unroll
  for (int piece = 0; piece < 3; ++piece) {
    const uint32_t ta = __float_as_uint(a) & 0xFFFF0000u, tb = __float_as_uint(b) & 0xFFFF0000u;
    sink(piece, ta >> 16 | tb);
    a -= __uint_as_float(ta);
    b -= __uint_as_float(tb);
  }
}

template <typename T>
__device__ __forceinline__ void store4(T* p, f32x4_t x) {
  if constexpr (sizeof(T) == 4) *reinterpret_cast<f32x4_t*>(p) = x;
  else *reinterpret_cast<u32x2_t*>(p) = u32x2_t{pack2<T>(x[0], x[1]), pack2<T>(x[2], x[3])};
}

template <typename T, int D>
__global__ __launch_bounds__(64) __attribute__((amdgpu_waves_per_eu(sizeof(T) == 4 ? 2 : 3))) void
paged_decode_q8_mfma_kernel(DecodeQ8Args a) {
  constexpr int KCH = D / 16;        // 16-byte chunks per row
  constexpr int RPI = 64 / KCH;      // rows per load instruction (8 or 16)
  constexpr int IPS = 16 / RPI;      // load instructions per 16-token step
  constexpr int NI = 2 * IPS;        // per chunk, K and V each
  constexpr int KC = D / 64;         // LDS reads per 16 tokens of K
  constexpr int DT = D / 16;         // 16-dim tiles of O^T
  constexpr int kStage = 2 * kChunk * D;
  constexpr bool kF16 = std::is_same<T, f16_t>::value;
  constexpr int kPieces = sizeof(T) == 4 ? 3 : 1;
  __shared__ __attribute__((aligned(256))) uint8_t stage[kStages * kStage + 4 * kSegment];
  const int lane = threadIdx.x;
  const int col = lane & 15, grp = lane >> 4;
  const int bs = a.d.block_size, sh = a.d.bs_shift;

  const uint32_t first = blockIdx.x / (uint32_t)a.units, next = gridDim.x / (uint32_t)a.units;
  const int unit = (int)(blockIdx.x - first * (uint32_t)a.units);
  const int kvh = a.tiles == 1 ? unit : unit / a.tiles;
  const int head0 = kvh * a.d.group + (unit - kvh * a.tiles) * 16;
  const int heads = min(16, (kvh + 1) * a.d.group - head0);
  const bool hcol = col < heads;
  const uint8_t* kbase = reinterpret_cast<const uint8_t*>(a.d.k) + (int64_t)kvh * a.d.k_head;
  const uint8_t* vbase = reinterpret_cast<const uint8_t*>(a.d.v) + (int64_t)kvh * a.d.v_head;
  const uint8_t* sbase = a.scales + (int64_t)kvh * a.s_head;
  const uint32_t lds0 = lds_offset(stage);
  const uint32_t lds_sc = lds0 + kStages * kStage;

  // This lane's byte offset of load instruction r of a chunk from its 16-token step's
  // first row: row RPI r + lane / KCH of the chunk, chunk by the row's swizzle.
  const int lrow = lane / KCH;
  uint32_t loff[NI];
#pragma unroll
  for (int r = 0; r < NI; ++r)
    loff[r] = (uint32_t)((RPI * r + lrow) & 15) * (uint32_t)a.d.k_token +
              16 * ((lane % KCH) ^ q8_swizzle<D>(RPI * r + lrow));
  // LDS byte offsets of the operand reads.
  uint32_t koff[2][KC], voff[DT];
#pragma unroll
  for (int t = 0; t < 2; ++t)
#pragma unroll
    for (int c = 0; c < KC; ++c)
      koff[t][c] = lds0 + (16 * t + col) * D + ((16 * (grp ^ q8_swizzle<D>(16 * t + col))) ^ (64 * c));
  const int vrow = (col >> 1) < 4 ? 4 * grp + (col >> 1) : 12 + 4 * grp + (col >> 1);
#pragma unroll
  for (int t = 0; t < DT; ++t)
    voff[t] = lds0 + kChunk * D + vrow * D + ((16 * q8_swizzle<D>(vrow)) ^ (16 * t)) + 8 * (col & 1);

  WalkQ8 walk;
  q8_start(a, first, walk);
  ItemQ8 it;
  while (q8_next(a, next, walk, it)) {
    const int n = it.n;
    T* out = reinterpret_cast<T*>(a.d.out) + it.qrow * a.d.o_row + (int64_t)(head0 + col) * a.d.o_head + 4 * grp;
    if (n <= 0) {
      if (n == 0 && it.split == 0 && hcol) {
#pragma unroll
        for (int t = 0; t < DT; ++t) store4(out + 16 * t, f32x4_t{0.f, 0.f, 0.f, 0.f});
      }
      continue;
    }
    const PartitionQ8 P = partition_q8(n, a);
    if (it.split >= P.nsplit) continue;
    const int s0 = P.first + it.split * P.bps;
    const int s1 = min(s0 + P.bps, P.first + P.pages);
    const int32_t* table = a.d.tables + it.trow * a.d.table_stride;
    // The first page ids travel with the queries.
    int ids = s0 + lane < min(s1, s0 + kSegment) ? table[s0 + lane] : 0;

    // Q^T operands of k-step (c, i): dims 64 c + 16 grp + 8 i .. + 7.
    u32x4_t qop[KC][2][kPieces];
    {
      const T* qp = reinterpret_cast<const T*>(a.d.q) + it.qrow * a.d.q_row +
                    (int64_t)(head0 + (hcol ? col : 0)) * a.d.q_head + 16 * grp;
#pragma unroll
      for (int c = 0; c < KC; ++c)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          constexpr int W = (int)sizeof(T) / 2;  // 16-byte loads
          u32x4_t x[W];
#pragma unroll
          for (int w = 0; w < W; ++w) {
            x[w] = *reinterpret_cast<const u32x4_t*>(qp + 64 * c + 8 * i + 4 * w);
            x[w] = hcol ? x[w] : u32x4_t{0u, 0u, 0u, 0u};
          }
          if constexpr (kPieces == 1) {
            qop[c][i][0] = x[0];
          } else {
#pragma unroll
            for (int w = 0; w < 4; ++w)
              split3(__uint_as_float(x[w / 2][2 * w % 4]), __uint_as_float(x[w / 2][2 * w % 4 + 1]),
                     [&](int piece, uint32_t pair) { qop[c][i][piece][w] = pair; });
          }
        }
    }

    float m = -1e30f, lsum = 0.f;  // of this lane's head column; lsum over its token slots
    f32x4_t acc[DT];
#pragma unroll
    for (int t = 0; t < DT; ++t) acc[t] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    for (int seg = s0; seg < s1; seg += kSegment) {
      const int seg1 = min(s1, seg + kSegment);
      if (seg > s0) ids = seg + lane < seg1 ? table[seg + lane] : 0;
      const int blk = pool_block(ids, a);
      // The pages' exponents: the aligned word around each pair.
      const uint8_t* sp = sbase + (int64_t)blk * a.s_block;
      lds_dma4((const void*)((uintptr_t)sp & ~(uintptr_t)3), __builtin_amdgcn_readfirstlane(lds_sc));
      const uint64_t at = (uint64_t)(uint32_t)blk * (uint64_t)a.d.k_block;
      const int at_lo = (int)at, at_hi = (int)(at >> 32);
      const int t0 = seg << sh;  // first token of the segment
      const int tb = max(P.start, t0);
      const int te = (int)min((int64_t)n, (int64_t)seg1 << sh);
      // Chunk j holds tokens t0 + 32 j ..; those before the window's are not read.
      const int j0 = (tb - t0) / kChunk, j1 = (te - t0 + kChunk - 1) / kChunk;

      auto load = [&](int j, auto st_c) __attribute__((always_inline)) {
        constexpr int st = decltype(st_c)::value;
        const int p0 = j * kChunk;  // from t0
        const uint32_t kl = lds0 + st * kStage, vl = kl + kChunk * D;
        if (t0 + p0 >= tb && te - t0 - p0 >= kChunk) {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int page = (p0 + 16 * h) >> sh;
            const uint32_t row = (uint32_t)(p0 + 16 * h) & (uint32_t)(bs - 1);
            const uint64_t off = ((uint64_t)(uint32_t)__builtin_amdgcn_readlane(at_hi, page) << 32 |
                                  (uint32_t)__builtin_amdgcn_readlane(at_lo, page)) +
                                 (uint64_t)row * (uint32_t)a.d.k_token;
#pragma unroll
            for (int i = 0; i < IPS; ++i) {
              const int r = IPS * h + i;
              lds_stream16_s(kbase + off, loff[r], __builtin_amdgcn_readfirstlane(kl + 1024 * r));
              lds_stream16_s(vbase + off, loff[r], __builtin_amdgcn_readfirstlane(vl + 1024 * r));
            }
          }
          return;
        }
        // A chunk that reaches outside the visible tokens reads the nearest visible one
        // there: masked out of the softmax, and as finite as the row itself.
#pragma unroll 1
        for (int r = 0; r < NI; ++r) {
          const int i = RPI * r + lrow;
          const int pos = min(max(p0 + i, tb - t0), te - t0 - 1);
          const int64_t off = (int64_t)shfl_i32(blk, pos >> sh) * a.d.k_block +
                              (int64_t)(pos & (bs - 1)) * a.d.k_token +
                              16 * ((lane % KCH) ^ q8_swizzle<D>(i));
          lds_stream16(kbase + off, __builtin_amdgcn_readfirstlane(kl + 1024 * r));
          lds_stream16(vbase + off, __builtin_amdgcn_readfirstlane(vl + 1024 * r));
        }
      };
      // One page a lane, set when the exponents have landed: the factor of its scores,
      // and its V scale.
      float kf = 0.f, vf = 0.f, pf = 1.f;
      auto scales = [&]() {
        const uint32_t w = *reinterpret_cast<const uint32_t*>(stage + kStages * kStage + 4 * lane);
        const uint32_t e = ((uintptr_t)sp & 2) ? w >> 16 : w;
        // (0, of a page never written, would make NaN of masked scores)
        kf = q8_scale(max((int)(e & 255), kLeastExponent)) * a.d.scale_log2;
        v_scale<T>(e >> 8 & 255, vf, pf);
      };
      auto attend = [&](int j, auto st_c) __attribute__((always_inline)) {
        constexpr int st = decltype(st_c)::value;
        const int p0 = j * kChunk;
        f32x4_t sc[2];
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          sc[t] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int c = 0; c < KC; ++c) {
            const u32x4_t x = lds_read16(koff[t][c] + st * kStage);
            const u32x4_t lo = MfmaQ8<T>::widen(x[0], x[1], 1.f, 1.f);
            const u32x4_t hi = MfmaQ8<T>::widen(x[2], x[3], 1.f, 1.f);
#pragma unroll
            for (int w = 0; w < kPieces; ++w) {
              sc[t] = MfmaQ8<T>::run(lo, qop[c][0][w], sc[t]);
              sc[t] = MfmaQ8<T>::run(hi, qop[c][1][w], sc[t]);
            }
          }
        }
        // Scales of the chunk's two 16-token tiles (the second may lie past the last page).
        const int g0 = min(p0, te - t0 - 1) >> sh, g1 = min(p0 + 16, te - t0 - 1) >> sh;
        const float ks[2] = {readlane_f32(kf, g0), readlane_f32(kf, g1)};
        const float vs[2] = {readlane_f32(vf, g0), readlane_f32(vf, g1)};
        if (!(t0 + p0 >= tb && te - t0 - p0 >= kChunk)) {
          const int lo = tb - t0 - p0 - 4 * grp, hi = te - t0 - p0 - 4 * grp;
#pragma unroll
          for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i)
              sc[t][i] = 16 * t + i >= lo && 16 * t + i < hi ? sc[t][i] : -INFINITY;
        }
        float mx = fmaxf(fmaxf(fmaxf(sc[0][0], sc[0][1]), fmaxf(sc[0][2], sc[0][3])) * ks[0],
                         fmaxf(fmaxf(sc[1][0], sc[1][1]), fmaxf(sc[1][2], sc[1][3])) * ks[1]);
        // Over the four lane groups of the head column.
        {
          const auto x = __builtin_amdgcn_permlane32_swap(__float_as_uint(mx), __float_as_uint(mx), false, false);
          mx = fmaxf(__uint_as_float(x[0]), __uint_as_float(x[1]));
          const auto y = __builtin_amdgcn_permlane16_swap(__float_as_uint(mx), __float_as_uint(mx), false, false);
          mx = fmaxf(__uint_as_float(y[0]), __uint_as_float(y[1]));
        }
        // The reference moves only when a score passes it by more than kSlack, so that most
        // chunks leave the accumulators alone.
        if (__any(mx > m + Weights<T>::kSlack)) {
          const float top = fmaxf(m, mx - Weights<T>::kLift);
          const float corr = fast_exp2(m - top);
          lsum *= corr;
#pragma unroll
          for (int t = 0; t < DT; ++t) acc[t] *= corr;
          m = top;
        }
        float p[2][4];
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int i = 0; i < 4; ++i) p[t][i] = fast_exp2(fmaf(sc[t][i], ks[t], -m));
        lsum += ((p[0][0] + p[0][1]) + (p[0][2] + p[0][3])) + ((p[1][0] + p[1][1]) + (p[1][2] + p[1][3]));
        if constexpr (kF16) {
          const float ps[2] = {readlane_f32(pf, g0), readlane_f32(pf, g1)};
#pragma unroll
          for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) p[t][i] *= ps[t];
        }
        u32x4_t pop[kPieces];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if constexpr (kPieces == 1)
            pop[0][i] = pack2<T>(p[i / 2][2 * (i & 1)], p[i / 2][2 * (i & 1) + 1]);
          else
            split3(p[i / 2][2 * (i & 1)], p[i / 2][2 * (i & 1) + 1],
                   [&](int piece, uint32_t pair) { pop[piece][i] = pair; });
        }
#pragma unroll
        for (int t = 0; t < DT; ++t) {
          const u32x2_t x = lds_tr8(voff[t] + st * kStage);
          const u32x4_t v = MfmaQ8<T>::widen(x[0], x[1], vs[0], vs[1]);
#pragma unroll
          for (int w = 0; w < kPieces; ++w) acc[t] = MfmaQ8<T>::run(v, pop[w], acc[t]);
        }
      };
      // Step j: chunk j has landed (only the loads of later chunks may be in flight); the
      // stage of j - 1, whose reads have returned, takes chunk j + kStages - 1.
      auto step = [&](int j, auto now_c) __attribute__((always_inline)) {
        constexpr int now = decltype(now_c)::value;
        const int later = min(kStages - 2, j1 - 1 - j);
        if (kStages > 3 && later == 2) wait_loads<4 * NI>();
        else if (kStages > 2 && later == 1) wait_loads<2 * NI>();
        else wait_loads<0>();
        if (j == j0) scales();
        if (j + kStages - 1 < j1) load(j + kStages - 1, std::integral_constant<int, (now + kStages - 1) % kStages>{});
        attend(j, now_c);
        wait_lds();
      };
      static_assert(kStages >= 2 && kStages <= 4, "the waits above");
      auto each_stage = [&](auto f) __attribute__((always_inline)) {
        f(std::integral_constant<int, 0>{});
        f(std::integral_constant<int, 1>{});
        if constexpr (kStages > 2) f(std::integral_constant<int, 2>{});
        if constexpr (kStages > 3) f(std::integral_constant<int, 3>{});
      };
      each_stage([&](auto st) __attribute__((always_inline)) {
        if (decltype(st)::value < kStages - 1 && j0 + decltype(st)::value < j1) load(j0 + decltype(st)::value, st);
      });
      for (int j = j0; j < j1; j += kStages)
        each_stage([&](auto st) __attribute__((always_inline)) {
          if (j + decltype(st)::value < j1) step(j + decltype(st)::value, st);
        });
    }
    lsum += shfl_xor_f32(lsum, 16);
    lsum += shfl_xor_f32(lsum, 32);
    if (!hcol) continue;
    if (P.nsplit == 1) {
      const float inv = 1.f / lsum;
#pragma unroll
      for (int t = 0; t < DT; ++t)
        store4(out + 16 * t, acc[t] * inv);
      continue;
    }
    const int64_t idx = (it.row * a.d.q_heads + head0 + col) * a.slots + it.split;
    if (grp == 0) {
      a.d.part_ml[idx * 2] = m;
      a.d.part_ml[idx * 2 + 1] = lsum;
    }
    float* dst = a.d.part_acc + idx * D + 4 * grp;
#pragma unroll
    for (int t = 0; t < DT; ++t) *reinterpret_cast<f32x4_t*>(dst + 16 * t) = acc[t];
  }
}

template <typename T, int ND, int WAVES>
__global__ __launch_bounds__(256) void merge_q8_kernel(DecodeQ8Args a) {
  merge_q8<T, ND, WAVES>(a, blockIdx.x, a.d.row_base + blockIdx.y);
}

template <typename T>
void launch_valu(bool wide16, bool wide4, unsigned waves, hipStream_t s, const DecodeQ8Args& a) {
  if (wide16 && a.d.head_dim <= 64)
    hipLaunchKernelGGL((paged_decode_q8_kernel<T, 16, 4, 1>), dim3(waves), dim3(64), 0, s, a);
  else if (wide16 && a.d.head_dim <= 128)
    hipLaunchKernelGGL((paged_decode_q8_kernel<T, 16, 8, 1>), dim3(waves), dim3(64), 0, s, a);
  else if (wide16)
    hipLaunchKernelGGL((paged_decode_q8_kernel<T, 16, 16, 1>), dim3(waves), dim3(64), 0, s, a);
  else if (wide4)
    hipLaunchKernelGGL((paged_decode_q8_kernel<T, 4, 64, 1>), dim3(waves), dim3(64), 0, s, a);
  else
    hipLaunchKernelGGL((paged_decode_q8_kernel<T, 1, 64, 4>), dim3(waves), dim3(64), 0, s, a);
}

template <typename T, int ND>
void launch_merge_nd(unsigned rows, hipStream_t s, const DecodeQ8Args& a) {
  static_assert(kMaxSplitsQ8 <= 4 * kGroup, "groups of a row");
  if (a.slots <= kGroup)
    hipLaunchKernelGGL((merge_q8_kernel<T, ND, 1>), dim3((unsigned)ceil_div(a.d.q_heads, 4), rows), dim3(256), 0, s, a);
  else
    hipLaunchKernelGGL((merge_q8_kernel<T, ND, 4>), dim3((unsigned)a.d.q_heads, rows), dim3(256), 0, s, a);
}

template <typename T>
void launch_merge_q8(unsigned rows, hipStream_t s, const DecodeQ8Args& a) {
  if (a.d.head_dim <= 64) launch_merge_nd<T, 1>(rows, s, a);
  else if (a.d.head_dim <= 128) launch_merge_nd<T, 2>(rows, s, a);
  else launch_merge_nd<T, 4>(rows, s, a);
}

template <typename T>
void launch_mfma_q8(unsigned groups, hipStream_t s, const DecodeQ8Args& a) {
  if (a.d.head_dim == 128)
    hipLaunchKernelGGL((paged_decode_q8_mfma_kernel<T, 128>), dim3(groups), dim3(64), 0, s, a);
  else
    hipLaunchKernelGGL((paged_decode_q8_mfma_kernel<T, 64>), dim3(groups), dim3(64), 0, s, a);
}

// Pages that a row of this table (and window) can touch, and the splits they make.
int64_t most_pages(int32_t table_width, int32_t block_size, int32_t window) {
  const int64_t pages = window > 0 ? std::min<int64_t>(table_width, (int64_t)window / block_size + 2) : table_width;
  return std::max<int64_t>(1, pages);
}
int split_pages(int32_t tokens, int32_t block_size) { return std::max(1, tokens / block_size); }
int most_splits_q8(int32_t table_width, int32_t block_size, int32_t window) {
  const int64_t pages = most_pages(table_width, block_size, window);
  const int64_t short_pages = std::min<int64_t>(pages, kShortTokens / block_size);
  int64_t most = std::max<int64_t>(1, ceil_div64(short_pages, split_pages(kSplitTokens, block_size)));
  if (pages > short_pages) most = std::max(most, ceil_div64(pages, split_pages(kLongTokens, block_size)));
  return (int)std::min<int64_t>(kMaxSplitsQ8, most);
}

size_t ml_bytes(int64_t slots) { return ((size_t)slots * 2 * sizeof(float) + 255) & ~(size_t)255; }

}  // namespace
}  // namespace vrh

using namespace vrh;

extern "C" size_t vrh_paged_decode_q8_workspace_bytes(int64_t rows, int32_t q_heads, int32_t head_dim,
                                                      int32_t block_size, int32_t table_width,
                                                      int32_t window) {
  if (rows <= 0 || q_heads <= 0 || head_dim <= 0 || block_size <= 0 || table_width < 0 || window < 0) return 0;
  const int splits = most_splits_q8(table_width, block_size, window);
  if (splits <= 1) return 0;
  const int64_t slots = rows * q_heads * splits;
  return ml_bytes(slots) + (size_t)slots * head_dim * sizeof(float);
}

int vrh_decode_rows_q8(const Q8Call& c, const int32_t* cu_q, int32_t num_seqs, int32_t expand_e,
                       int64_t rows, int32_t window, void* workspace, size_t workspace_bytes,
                       bool one_split, hipStream_t s, const char* who, DecodeQ8Args* later,
                       unsigned* later_blocks) {
  const int es = dtype_bytes(c.dtype);
  VRH_CHECK_ARG(es > 0, "%s: unknown dtype %d", who, c.dtype);
  VRH_CHECK_ARG(rows >= 0 && c.q_heads >= 1 && c.kv_heads >= 1 && c.q_heads % c.kv_heads == 0,
                "%s: query heads must be a positive multiple of KV heads", who);
  VRH_CHECK_ARG(c.q_heads <= 65535, "%s: too many heads", who);
  VRH_CHECK_ARG(c.head_dim >= 1 && c.head_dim <= 256, "%s: head_dim %d unsupported", who, c.head_dim);
  VRH_CHECK_ARG(c.block_size >= 1 && c.table_width >= 0 && window >= 0 && c.num_blocks >= 1,
                "%s: bad block_size/table_width/window/num_blocks", who);
  if (rows == 0) return VRH_OK;
  VRH_CHECK_ARG(c.out && c.q && c.k && c.v && c.scales && c.lengths && (c.tables || c.table_width == 0),
                "%s: null pointer", who);
  DecodeQ8Args a = {};
  a.scales = (const uint8_t*)c.scales;
  a.s_block = c.s_block;
  a.s_head = c.s_head;
  a.num_blocks = c.num_blocks;
  a.slots = one_split ? 1 : most_splits_q8(c.table_width, c.block_size, window);
  const int64_t slots = rows * c.q_heads * a.slots;
  if (a.slots > 1) {
    const size_t need = ml_bytes(slots) + (size_t)slots * c.head_dim * sizeof(float);
    VRH_CHECK_ARG(workspace && workspace_bytes >= need, "%s: workspace of %zu bytes needed, %zu given", who,
                  need, workspace ? workspace_bytes : (size_t)0);
    VRH_CHECK_ARG(((uintptr_t)workspace & 255) == 0, "%s: workspace misaligned", who);
    a.d.part_ml = (float*)workspace;
    a.d.part_acc = (float*)((char*)workspace + ml_bytes(slots));
  }
  a.d.out = c.out;
  a.d.q = c.q;
  a.d.k = c.k;
  a.d.v = c.v;
  a.d.tables = c.tables;
  a.d.lengths = c.lengths;
  a.d.rows = rows;
  a.d.q_row = c.q_row;
  a.d.q_head = c.q_head;
  a.d.o_row = c.o_row;
  a.d.o_head = c.o_head;
  a.d.k_block = a.d.v_block = c.c_block;
  a.d.k_token = a.d.v_token = c.c_token;
  a.d.k_head = a.d.v_head = c.c_head;
  a.d.table_stride = c.table_stride;
  a.d.cu_q = cu_q;
  a.d.num_seqs = num_seqs;
  a.d.expand_e = expand_e;
  a.d.q_heads = c.q_heads;
  a.d.group = c.q_heads / c.kv_heads;
  a.d.head_dim = c.head_dim;
  a.d.block_size = c.block_size;
  a.d.bs_shift = (c.block_size & (c.block_size - 1)) == 0 ? __builtin_ctz((unsigned)c.block_size) : -1;
  a.d.window = window;
  a.d.min_bps = split_pages(kSplitTokens, c.block_size);
  a.d.long_bps = split_pages(kLongTokens, c.block_size);
  a.d.short_pages = kShortTokens / c.block_size;
  a.d.table_width = c.table_width;
  a.d.scale_log2 = (float)(1.4426950408889634 / std::sqrt((double)c.head_dim));
  auto cache_aligned = [&](int v) {
    return c.head_dim % v == 0 && c.c_block % v == 0 && c.c_token % v == 0 && c.c_head % v == 0 &&
           (uintptr_t)c.k % v == 0 && (uintptr_t)c.v % v == 0;
  };
  // The matrix kernel: head_dim 64 or 128, blocks of a power of two of
  // tokens from 16 on, 16-byte aligned rows, scale pairs that do not straddle a word, row offsets
  // within a load instruction in 32 bits.
  const bool mfma = (c.head_dim == 64 || c.head_dim == 128) &&
                    a.d.bs_shift >= 4 && c.block_size <= 65536 && cache_aligned(16) && c.c_token < (1 << 26) &&
                    c.c_token >= 0 && c.c_block >= 0 && c.q_row * es % 16 == 0 &&
                    c.q_head * es % 16 == 0 && c.o_row % 4 == 0 && c.o_head % 4 == 0 &&
                    (uintptr_t)c.q % 16 == 0 && (uintptr_t)c.out % (4 * es) == 0 && c.s_block % 2 == 0 && c.s_head % 2 == 0 &&
                    (uintptr_t)c.scales % 2 == 0;
  a.tiles = mfma ? ceil_div(a.d.group, 16) : 1;
  a.units = mfma ? c.kv_heads * a.tiles : c.q_heads;
  auto shift_of = [](int x) { return (x & (x - 1)) == 0 ? __builtin_ctz((unsigned)x) : -1; };
  a.min_shift = shift_of(a.d.min_bps);
  a.long_shift = shift_of(a.d.long_bps);
  a.split_unit = mfma ? std::max(1, kChunk / c.block_size) : 1;
  a.compact = rows <= kCompactRows;
  const int64_t per_row = (int64_t)a.units * a.slots;
  // A launch has less than 2^32 threads (65535 heads of kMaxSplitsQ8 splits at most, so at
  // least one row); the waves that share the splits are fewer, and walk all rows.
  const int64_t kRowsPerLaunch =
      a.compact ? rows : std::min<int64_t>(65535, ((1ll << 26) - 1) / per_row);
  // Waves that are resident at once: by LDS, or of the VALU kernel by registers.
  constexpr int64_t kCus = 256, kLds = 160 * 1024;
  const int64_t resident = kCus * (mfma ? kLds / (kStages * 2 * kChunk * c.head_dim + 1024) : 12);
  for (int64_t first = 0; first < rows; first += kRowsPerLaunch) {
    a.d.row_base = first;
    const unsigned count = (unsigned)std::min<int64_t>(rows - first, kRowsPerLaunch);
    int64_t waves = count * per_row;
    if (a.compact) waves = std::min(waves, std::max<int64_t>(1, resident / a.units) * a.units);
    // The caller merges the rows with its own partials.
    const bool defer = later != nullptr && a.slots > 1 && count == rows;
    if (defer) {
      *later = a;
      *later_blocks = (unsigned)(ceil_div(c.q_heads * (a.slots <= kGroup ? 1 : 4), 4) * rows);
    }
    const bool merge = a.slots > 1 && !defer;
    switch (c.dtype) {
      case VRH_DTYPE_F32:
        if (mfma) launch_mfma_q8<float>((unsigned)waves, s, a);
        else launch_valu<float>(cache_aligned(16), cache_aligned(4), (unsigned)waves, s, a);
        if (merge) launch_merge_q8<float>(count, s, a);
        break;
      case VRH_DTYPE_F16:
        if (mfma) launch_mfma_q8<f16_t>((unsigned)waves, s, a);
        else launch_valu<f16_t>(cache_aligned(16), cache_aligned(4), (unsigned)waves, s, a);
        if (merge) launch_merge_q8<f16_t>(count, s, a);
        break;
      default:
        if (mfma) launch_mfma_q8<bf16_t>((unsigned)waves, s, a);
        else launch_valu<bf16_t>(cache_aligned(16), cache_aligned(4), (unsigned)waves, s, a);
        if (merge) launch_merge_q8<bf16_t>(count, s, a);
    }
  }
  VRH_RETURN_LAUNCH(who);
}

extern "C" int vrh_paged_decode_q8(int dtype, void* out, const void* q, const void* key_cache,
                                   const void* value_cache, const void* scales,
                                   const int32_t* block_tables, const int32_t* context_lengths,
                                   int64_t rows, int32_t q_heads, int32_t kv_heads, int32_t head_dim,
                                   int64_t num_blocks, int32_t block_size, int32_t table_width,
                                   int64_t table_stride, int64_t q_row_stride, int64_t q_head_stride,
                                   int64_t out_row_stride, int64_t out_head_stride,
                                   int64_t cache_block_stride, int64_t cache_token_stride,
                                   int64_t cache_head_stride, int64_t scale_block_stride,
                                   int64_t scale_head_stride, int32_t window, void* workspace,
                                   size_t workspace_bytes, vrh_stream_t stream) {
  const Q8Call c = {dtype, out, q, key_cache, value_cache, scales, block_tables, context_lengths,
                    q_heads, kv_heads, head_dim, num_blocks, block_size, table_width, table_stride,
                    q_row_stride, q_head_stride, out_row_stride, out_head_stride, cache_block_stride,
                    cache_token_stride, cache_head_stride, scale_block_stride, scale_head_stride};
  return vrh_decode_rows_q8(c, nullptr, 0, 0, rows, window, workspace, workspace_bytes, false,
                            (hipStream_t)stream, "vrh_paged_decode_q8");
}
