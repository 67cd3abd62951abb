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

// Decode rows (the rows of cu_q / expand_e: see DecodeArgs). With one_split every row
// is one split and needs no workspace.
int vrh_decode_rows_q8(const Q8Call& c, const int32_t* cu_q, int32_t num_seqs, int32_t expand_e,
                       int64_t rows, int32_t window, void* workspace, size_t workspace_bytes,
                       bool one_split, hipStream_t s, const char* who);

namespace vrh {

struct DecodeQ8Args {
  DecodeArgs d;  // K and V strides in bytes; part_ml, part_acc [rows, q_heads, slots, ..]
  const uint8_t* scales;
  int64_t s_block, s_head;
  int64_t num_blocks;
  int32_t slots;  // most splits of a row
};

// A page id brought into the pool: an id that is not one of its blocks (a caller's
// mistake) reads some block instead of memory outside the pool.
__device__ __forceinline__ int pool_block(int id, const DecodeQ8Args& a) {
  return (int)max((int64_t)0, min((int64_t)id, a.num_blocks - 1));
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

}  // namespace vrh
