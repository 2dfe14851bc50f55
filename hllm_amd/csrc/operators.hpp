// Launchers of the operators on device memory (operators.hip). Arguments are checked by the C
// entry points; every launch goes to `stream` on the current device.
#pragma once

#include <cstdlib>
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
  uint32_t page_stride, token_stride;  // bytes
  uint64_t head_stride;
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
  int32_t blocks;                // workgroups
  int32_t shared;                // the rows' work is cut into the workgroups' shares (else a pair each)
  float scale_hi, scale_lo;      // the scores' scale times log2 e as a sum of two floats
  int2* cuts;                    // [pairs]: the first workgroup and the number of its parts (null: no pair is cut)
  float* part;                   // [blocks][2][min(group, 16)][D]: parts' outputs, each normalised
  float* stats;                  // [blocks][2][min(group, 16)][2]: their score maximum (base 2) and sum
};
void launch_kv_attention(hipStream_t stream, uint32_t dtype, int format, int head_dim, const AttendArgs& a);

// Steps (of 128 positions) that starting a pair is counted as. With 1, 2, 3, 4: 128 rows to 8192 positions of head dimension
// 256 52.8, 52.7, 53.7, 55.2 us; 32 rows to 4096 of 64 14.6, 15.0, 16.0, 16.1; 64 rows to 8192 of 128 43.5, 43.9, 44.1,
// 44.9; 16 rows to 2048 of 128 13.6, 13.2, 13.4, 14.2.
constexpr int kPairCost = 1;
// Rows whose lengths every workgroup sums to find its share: sixteen a lane. Past them every pair is whole: a row of 32000
// positions takes 79 us among 1024 rows of 40, 296 among 1025; rows log-uniform to 8192 539 and 541.
constexpr uint64_t kMostSharedRows = 1024;
// Workgroups that the card's 256 CUs hold at once, by LDS (a wave's tile) and registers (about a hundred and
// D / 2); F32 queries of 256 elements leave room for one on a CU.
template <int D>
constexpr int kAttendBlocks = D == 64 ? 4 : D == 128 ? 3 : 2;
inline uint64_t attend_blocks(int head_dim, bool f32) {
  return 256 * (head_dim == 64 ? kAttendBlocks<64> : head_dim == 128 ? kAttendBlocks<128> : f32 ? 1 : kAttendBlocks<256>);
}

}  // namespace hllm_rocm
