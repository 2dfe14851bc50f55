// Launchers of the operators on device memory (operators.hip). Arguments are checked by the C
// entry points; every launch goes to `stream` on the current device.
#pragma once

#include "common.hpp"

namespace hllm_rocm {

// A tensor [rows][heads][D] as kernels take it: strides in elements.
struct Strided {
  void* data;
  uint64_t row, head;
};

// A cache as kernels take it; a slot is page << page_shift | position.
struct Pages {
  uint8_t* keys;
  uint8_t* values;
  float* key_scales;
  float* value_scales;
  uint64_t page_stride, token_stride, head_stride;  // bytes
  int32_t pages, page_shift, kv_heads;
};

struct RotateArgs {
  Strided q, q_out, k, k_out, v;
  int32_t q_heads, k_heads, v_heads;
  int32_t lanes;           // lanes of a head: D / 16
  int32_t heads_per_block;
  const int32_t* positions;
  const int32_t* slots;    // append
  Pages pages;             // append
  int32_t rotary;          // rotated elements (0: none)
  int32_t interleaved;
  float magnitude;
  uint64_t turns[128];
};
// q and k rotated into q_out and k_out (format -1), or k rotated and k and v quantised into the
// cache (format: hllm_kv_format).
void launch_rotate(hipStream_t stream, uint32_t dtype, int format, int rows, const RotateArgs& a);

struct ReadArgs {
  Pages pages;
  const int32_t* slots;
  Strided k, v;
  int32_t rows;
};
void launch_kv_read(hipStream_t stream, uint32_t dtype, int format, int head_dim, const ReadArgs& a);

struct AttendArgs {
  Pages pages;
  Strided q, out;
  const int32_t* table;
  uint64_t table_stride;
  const int32_t* lengths;
  int32_t rows, q_heads, group;  // group: query heads of one KV head
  int32_t head_groups;           // sixteens of a KV head's query heads
  int32_t limit;                 // positions of a row that count at most
  int32_t splits, unit;          // attend_split
  float scale;
  float* part;                   // [rows][q_heads][splits][D]: splits' outputs, each normalised
  float* stats;                  // [rows][q_heads][splits][2]: their score maximum (base 2) and sum
};
void launch_kv_attention(hipStream_t stream, uint32_t dtype, int format, int head_dim, const AttendArgs& a);

// Positions that one workgroup holds page numbers for.
constexpr int kAttendMostKeys = 8192;
// How a call splits its rows: at most `splits` parts of a row, of at least `unit` positions.
struct AttendSplit {
  int splits, unit;
};
// `pairs`: rows x KV heads x sixteens of query heads.
inline AttendSplit attend_split(uint64_t pairs, uint64_t limit) {
  constexpr uint64_t kTarget = 2048, kUnit = 128;
  const uint64_t wanted = (kTarget + pairs - 1) / pairs, most = (limit + kUnit - 1) / kUnit;
  const uint64_t least = (limit + kAttendMostKeys - 1) / kAttendMostKeys;
  uint64_t splits = wanted < most ? wanted : most;
  if (splits < least) splits = least;
  if (splits < 1) splits = 1;
  return {(int)splits, (int)kUnit};
}
// Positions of each part of a row of `length`: a multiple of 32.
__host__ __device__ inline int attend_part(int length, int splits, int unit) {
  const int per = (int)(((int64_t)length + splits - 1) / splits);
  return ((per > unit ? per : unit) + 31) & ~31;
}

}  // namespace hllm_rocm
