// What the decode and prefill of the 8-bit cache share: a call's arguments and the
// decode rows' launcher.
#pragma once

#include "decode_rows.h"
#include "q8.h"

// Arguments of an attention call over the 8-bit cache (strides in elements; the
// cache's elements are bytes).
struct Q8Call {
  int dtype;
  void* out;
  const void* q;
  const void* k;
  const void* v;
  const void* scales;
  const int32_t* tables;
  const int32_t* lengths;
  int32_t q_heads, kv_heads, head_dim;
  int64_t num_blocks;
  int32_t block_size, table_width;
  int64_t table_stride;
  int64_t q_row, q_head, o_row, o_head;
  int64_t c_block, c_token, c_head;
  int64_t s_block, s_head;
};

namespace vrh {

struct DecodeQ8Args {
  DecodeArgs d;  // K and V strides in bytes; part_ml, part_acc [rows, q_heads, slots, ..]
  const uint8_t* scales;
  int64_t s_block, s_head;
  int64_t num_blocks;
  int32_t slots;  // most splits of a row
  int32_t tiles;  // waves of up to 16 q heads per KV head (MFMA kernel)
  int32_t units;  // kv_heads * tiles
  int32_t compact;  // waves share the splits that exist (MFMA kernel)
  int32_t split_unit;  // splits are whole multiples of this many pages (a power of two)
  int32_t min_shift;   // log2 of d.min_bps, a short row's pages per split, or -1
  int32_t long_shift;  // log2 of d.long_bps, a longer row's, or -1
};

// A page id brought into the pool: an id that is not one of its blocks (a caller's
// mistake) reads some block instead of memory outside the pool.
__device__ __forceinline__ int pool_block(int id, const DecodeQ8Args& a) {
  return (int)max((int64_t)0, min((int64_t)id, a.num_blocks - 1));
}

// Splits of rows of up to kShortTokens visible tokens and of longer ones, and the most
// splits of a row. Long rows come in batches or are cut into many splits anyway, and a
// split costs a wave's start and a partial: 64 rows of 512-4096 tokens (16 x 128 heads)
// 113 us with splits of 128 tokens throughout, 107 with 256; 512 no better. Short rows
// are what few waves have: one row of 300 tokens in three splits.
constexpr int kSplitTokens = 128;
constexpr int kLongTokens = 256;  // (37 float16 rows, 32 over 8 heads: 48 us, 61 with 128, 55 with 512)
constexpr int kShortTokens = 2048;
constexpr int kMaxSplitsQ8 = 64;  // a lane each in the merge

struct PartitionQ8 {
  int start;   // first visible token
  int first;   // first page
  int pages;   // pages touched
  int bps;     // pages per split
  int nsplit;
};

__device__ __forceinline__ PartitionQ8 partition_q8(int n, const DecodeQ8Args& a) {
  PartitionQ8 p;
  p.start = (a.d.window > 0 && n > a.d.window) ? n - a.d.window : 0;
  if (a.d.bs_shift >= 0) {
    p.first = p.start >> a.d.bs_shift;
    p.pages = ((n - 1) >> a.d.bs_shift) + 1 - p.first;
  } else {
    p.first = p.start / a.d.block_size;
    p.pages = (n - 1) / a.d.block_size + 1 - p.first;
  }
  // Fewer slots than the most splits: the table (or window) has no longer rows, or one
  // split is asked for.
  if (a.slots == 1) {
    p.bps = (p.pages + a.split_unit - 1) & -a.split_unit;
    p.nsplit = 1;
  } else {
    const bool longer = p.pages > a.d.short_pages;
    const int shift = longer ? a.long_shift : a.min_shift;
    if (shift >= 0 && p.pages <= kMaxSplitsQ8 << shift) {
      p.bps = 1 << shift;  // (no division: a wave does this before its first load)
      p.nsplit = (p.pages + p.bps - 1) >> shift;
    } else {
      p.bps = max(longer ? a.d.long_bps : a.d.min_bps, (p.pages + kMaxSplitsQ8 - 1) / kMaxSplitsQ8);
      p.bps = (p.bps + a.split_unit - 1) & -a.split_unit;
      p.nsplit = (int)((uint32_t)(p.pages + p.bps - 1) / (uint32_t)p.bps);
    }
  }
  return p;
}

// The partials of a (row, q head), ND dims a lane: up to kGroup splits by one wave, in
// split order with all loads in flight at once; more by WAVES waves, a group each, whose
// sums are added in order (so that the result does not depend on WAVES).
constexpr int kGroup = 16;
// Workgroups of 4 waves: `block` of the ceil(q_heads * WAVES / 4) of a row.
template <typename T, int ND, int WAVES>
__device__ __forceinline__ void merge_q8(const DecodeQ8Args& a, int block, int64_t row) {
  constexpr int kHeads = 4 / WAVES;  // of a workgroup
  const int lane = threadIdx.x & 63;
  const int wave = threadIdx.x >> 6;
  const int head = block * kHeads + wave / WAVES;
  const int group = wave % WAVES;
  if (head >= a.d.q_heads) return;
  int64_t trow, qrow;
  const int n = row_length(row, a.d, &trow, &qrow);
  if (n <= 0) return;
  const PartitionQ8 P = partition_q8(n, a);
  if (P.nsplit <= 1) return;
  const int64_t idx = (row * a.d.q_heads + head) * a.slots;
  const int s0 = kGroup * group;
  const float* src = a.d.part_acc + (idx + s0) * a.d.head_dim;
  float x[kGroup][ND];
#pragma unroll
  for (int u = 0; u < kGroup; ++u)
#pragma unroll
    for (int j = 0; j < ND; ++j) {
      const int d = lane + 64 * j;
      x[u][j] = s0 + u < P.nsplit && d < a.d.head_dim ? src[u * a.d.head_dim + d] : 0.f;
    }
  const float mi = lane < P.nsplit ? a.d.part_ml[(idx + lane) * 2] : -INFINITY;
  const float li = lane < P.nsplit ? a.d.part_ml[(idx + lane) * 2 + 1] : 0.f;
  const float M = wave_max(mi);
  const float wi = lane < P.nsplit ? fast_exp2(mi - M) : 0.f;
  const float inv = 1.f / wave_sum(wi * li);
  float acc[ND] = {};
#pragma unroll
  for (int u = 0; u < kGroup; ++u) {
    const float w = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(wi), s0 + u));
    if (s0 + u < P.nsplit) {
#pragma unroll
      for (int j = 0; j < ND; ++j) acc[j] = fmaf(w, x[u][j], acc[j]);
    }
  }
  if constexpr (WAVES > 1) {
    __shared__ float sums[WAVES][ND][64];
#pragma unroll
    for (int j = 0; j < ND; ++j) sums[group][j][lane] = acc[j];
    __syncthreads();
    if (group > 0) return;
    for (int g = 1; g * kGroup < P.nsplit; ++g)
#pragma unroll
      for (int j = 0; j < ND; ++j) acc[j] += sums[g][j][lane];
  }
  T* out = reinterpret_cast<T*>(a.d.out) + qrow * a.d.o_row + (int64_t)head * a.d.o_head;
#pragma unroll
  for (int j = 0; j < ND; ++j)
    if (lane + 64 * j < a.d.head_dim) out[lane + 64 * j] = from_f32<T>(acc[j] * inv);
}

// Scale exponents of one (page, head): K's in bits 0-7, V's in bits 8-15.
__device__ __forceinline__ uint32_t q8_exponents(const uint8_t* p) {
  return (uint32_t)p[0] | (uint32_t)p[1] << 8;
}

// VE e4m3 bytes to floats.
template <int VE>
__device__ __forceinline__ void q8_values(raw_of<VE> raw, float (&x)[VE]) {
  if constexpr (VE == 1) {
    x[0] = q8_to_f32(raw);
  } else {
    union {
      raw_of<VE> r;
      uint32_t w[VE / 4];
    } u;
    u.r = raw;
#pragma unroll
    for (int i = 0; i < VE; i += 4) {
      float f[4];
      q8_unpack4(u.w[i / 4], f);
#pragma unroll
      for (int j = 0; j < 4; ++j) x[i + j] = f[j];
    }
  }
}

// 16-bit operands of 8 e4m3 bytes, and the products they feed.
typedef __attribute__((ext_vector_type(8))) __bf16 q8_bf16x8;
typedef __attribute__((ext_vector_type(8))) _Float16 q8_f16x8;
typedef __attribute__((ext_vector_type(4))) float q8_f32x4;
typedef __attribute__((ext_vector_type(16))) float q8_f32x16;
typedef __attribute__((ext_vector_type(4))) uint32_t q8_u32x4;

template <typename T>
struct MfmaQ8;
template <>
struct MfmaQ8<bf16_t> {
  // Bytes 0-3 times s0, 4-7 times s1 (powers of two, exact).
  __device__ static q8_u32x4 widen(uint32_t lo, uint32_t hi, float s0, float s1) {
    return q8_u32x4{
        __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, s0, false)),
        __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, s0, true)),
        __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, s1, false)),
        __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, s1, true))};
  }
  __device__ static q8_f32x4 run(q8_u32x4 a, q8_u32x4 b, q8_f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(q8_bf16x8, a),
                                                   __builtin_bit_cast(q8_bf16x8, b), c, 0, 0, 0);
  }
};
template <>
struct MfmaQ8<float> : MfmaQ8<bf16_t> {};  // in bf16 pieces
template <>
struct MfmaQ8<f16_t> {
  __device__ static q8_u32x4 widen(uint32_t lo, uint32_t hi, float s0, float s1) {
    return q8_u32x4{
        __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, s0, false)),
        __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, s0, true)),
        __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, s1, false)),
        __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, s1, true))};
  }
  __device__ static q8_f32x4 run(q8_u32x4 a, q8_u32x4 b, q8_f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(q8_f16x8, a),
                                                  __builtin_bit_cast(q8_f16x8, b), c, 0, 0, 0);
  }
};

// Softmax weights are rounded to the query's type for the V product: exp2(s - m) where
// the reference m was the largest score minus kLift when it last moved, and moves when
// a score passes it by kSlack. bf16 rounds every weight by at most 2^-8 of it (half a step;
// float32 weights are split into exact pieces instead). f16 has
// few exponents: lifted by 2^7 its weights go down to 2^-21 of the largest before they
// get subnormal (2^-14 unlifted), and up to 2^12 (2^15 with the factor of v_scale).
template <typename T>
struct Weights {
  static constexpr float kLift = 0.f, kSlack = 8.f;
};
template <>
struct Weights<f16_t> {
  static constexpr float kLift = 7.f, kSlack = 12.f;
};

// How a page's V scale 2^(e - 127) meets the product: vs in the bytes' conversion, ps
// on the weights. bf16 holds e4m3 * 2^(e - 127) exactly. f16 does up to 2^7 (448 * 2^7
// = 57344); what a larger scale has over that goes to the weights. Below 2^-15 the
// conversion rounds to f16's least step, 2^-24, which the f16 output has as well.
template <typename T>
__device__ __forceinline__ void v_scale(int e, float& vs, float& ps) {
  if constexpr (sizeof(T) == 2 && !__is_same(T, bf16_t)) {
    vs = q8_scale(min(e, 134));
    ps = q8_scale(max(e - 134, 0) + 127);
  } else {
    vs = q8_scale(e);
    ps = 1.f;
  }
}

// The LDS-direct loads of common.h for bytes that are read once (see lds_dma16).
__device__ __forceinline__ void lds_stream16(const void* g, uint32_t m0) {
  asm volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %0, off nt" ::"v"(g), "{m0}"(m0) : "memory");
}
__device__ __forceinline__ void lds_stream16_s(const void* base, uint32_t lane_off, uint32_t m0) {
  asm volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %0, %1 nt" ::"v"(lane_off), "s"(base), "{m0}"(m0)
               : "memory");
}

// 16 bytes at an LDS byte offset.
__device__ __forceinline__ q8_u32x4 lds_read16(uint32_t offset) {
  return *(const q8_u32x4 __attribute__((address_space(3)))*)(uintptr_t)offset;
}

// s_waitcnt vmcnt(N) for N up to 63, and lgkmcnt(0) (gfx9 encoding).
template <int N>
__device__ __forceinline__ void wait_loads() {
  static_assert(N >= 0 && N < 64, "vmcnt");
  __builtin_amdgcn_s_waitcnt((N & 15) | (N >> 4) << 14 | 0x7 << 4 | 0xF << 8);
  asm volatile("" ::: "memory");
}
__device__ __forceinline__ void wait_lds() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(15 | 3 << 14 | 0x7 << 4);
}

}  // namespace vrh

// Decode rows (the rows of cu_q / expand_e: see DecodeArgs). With one_split every row
// is one split and needs no workspace. With `later`, rows that fit one launch may be left
// unmerged: *later_blocks > 0 workgroups of 4 waves, block b running merge_q8 of block
// b % B of row b / B, B = ceil(q_heads * WAVES / 4), are then the caller's to launch
// (WAVES: 1 with up to kGroup slots, otherwise 4).
int vrh_decode_rows_q8(const Q8Call& c, const int32_t* cu_q, int32_t num_seqs, int32_t expand_e,
                       int64_t rows, int32_t window, void* workspace, size_t workspace_bytes,
                       bool one_split, hipStream_t s, const char* who, vrh::DecodeQ8Args* later = nullptr,
                       unsigned* later_blocks = nullptr);
