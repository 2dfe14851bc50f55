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

// Formats of a cache's vectors: hllm_kv_format, then hllm_kv4_format.
constexpr int kE2m1 = 2 + HLLM_KV4_E2M1, kInt4 = 2 + HLLM_KV4_INT4;
inline bool four_bits(int format) { return format >= kE2m1; }

// A cache as kernels take it; a slot is page << page_shift | position.
struct Pages {
  uint8_t* keys;
  uint8_t* values;
  void* key_scales;  // F32 for each vector; of 4 bits for each 32 elements: bytes (E2M1), BF16 (INT4)
  void* value_scales;
  uint32_t page_stride, token_stride;  // bytes
  uint64_t head_stride;
  int32_t pages, page_shift, kv_heads;
};

// ... and as entry points do.
struct Cache {
  Pages pages;
  int format, head_dim;
  uint32_t page_tokens;
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
// cache.
void launch_rotate(hipStream_t stream, uint32_t dtype, int format, int rows, const RotateArgs& a);

struct ReadArgs {
  Pages pages;
  const int32_t* slots;
  Strided k, v;
  int32_t rows;
};
void launch_kv_read(hipStream_t stream, uint32_t dtype, int format, int head_dim, const ReadArgs& a);
void launch_kv4_read(hipStream_t stream, uint32_t dtype, int format, int head_dim, const ReadArgs& a);

struct AttendArgs {
  Pages pages;
  Strided q, out;
  const int32_t* table;
  uint64_t table_stride, table_head;  // entries from one row's, and one KV head's, pages to the next
  const int32_t* lengths;
  int32_t rows, q_heads, group;  // group: query heads of one KV head
  int32_t head_groups;           // sixteens of a KV head's query heads
  int32_t limit;                 // positions of a row that count at most
  int32_t blocks;                // workgroups
  int32_t cluster;               // pairs that follow one another and read the same cache lines; pairs are a multiple of it
  int32_t shared;                // the rows' work is cut into the workgroups' shares (else a pair each)
  float scale_hi, scale_lo;      // the scores' scale times log2 e as a sum of two floats
  int2* cuts;                    // [pairs]: the first workgroup and the number of its parts (null: no pair is cut)
  float* part;                   // [blocks][2][min(group, 16)][D]: parts' outputs, each normalised
  float* stats;                  // [blocks][2][min(group, 16)][2]: their score maximum (base 2) and sum
};
void launch_kv_attention(hipStream_t stream, uint32_t dtype, int format, int head_dim, const AttendArgs& a);
// Without the join.
void launch_kv4_attention(hipStream_t stream, uint32_t dtype, int format, int head_dim, const AttendArgs& a);

// What takes a page and KV head.
enum BoundsBy { kByWorkgroup, kByWave, kBySlot };
struct BoundsArgs {
  Pages pages;
  int8_t* codes;           // [pages][kv_heads][2][D]
  float* scales;           // [pages][kv_heads]
  const int32_t* table;
  uint64_t table_stride;
  const int32_t* starts;   // [rows]: the first position whose page is to be bounded
  const int32_t* lengths;  // [rows]
  int32_t rows, limit;
  int32_t places;          // pages of a row at most
  int32_t by;              // BoundsBy
};

struct SelectArgs {
  Strided q;
  const int8_t* codes;
  const float* scales;
  const int32_t* table;
  uint64_t table_stride;
  const int32_t* lengths;
  int32_t* selected;          // [rows][kv_heads][keep]
  int32_t* selected_lengths;  // [rows]
  uint32_t* keys;             // [rows][kv_heads][stride]: the pages' scores as ordered whole numbers
  uint64_t stride;
  int32_t rows, kv_heads, group, pages, page_shift;
  int32_t limit;              // positions of a row that count at most
  int32_t keep, first, last;
};

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
// Over a 4-bit cache. Positions of a wave's tile, of which there are two in LDS, and workgroups on a CU. Us with tiles of 64 and one
// buffer / 32 and two / 32 and one / 64 and two, 24 rows of 12000 to 30000 positions:
//   E2M1, 128: 98.5 / 96.0 / 100.5 / 101.2; INT4, 128: 131 / 120 / 130 / 124; E2M1, 64: 72.2 / 76.9 / 73.3 / 68.4;
//   E2M1, 256: 94.6 / 96.2 / 96.0 / 93.4; INT4, 256, F32: 255 / 213 / 254 / 214
template <int D>
constexpr int kAttend4Tile = D == 64 ? 64 : 32;
template <int D>
constexpr int kAttend4Blocks = D == 256 ? 2 : 3;
// Steps that starting a pair is counted as. With 1, 2, 3, 4: 16 rows of 2048 positions 21.2, 19.2, 20.2, 19.9 us; 32 rows of
// 2048 27.0, 24.6, 26.6, 25.9; 64 rows to 8192 33.4, 32.6, 32.2, 33.3; 128 rows to 8192 of 256 83.6, 84.0, 89.7, 95.8.
constexpr int kPair4Cost = 2;
// `large`: queries that leave room for one workgroup where heads are of 256 elements (F32; F16 beside an E2M1 cache, as two BF16 parts:
// 24 rows of 12000 to 30000 positions 120 us with shares for one, 128 with shares for two; 64 to 2048 27.2 and 32.5).
inline uint64_t attend_blocks(int format, int head_dim, bool large) {
  if (four_bits(format)) return 256 * (head_dim == 64 ? kAttend4Blocks<64> : head_dim == 128 ? kAttend4Blocks<128> : large ? 1 : kAttend4Blocks<256>);
  return 256 * (head_dim == 64 ? kAttendBlocks<64> : head_dim == 128 ? kAttendBlocks<128> : large ? 1 : kAttendBlocks<256>);
}
inline int attend_cost(int format) { return four_bits(format) ? kPair4Cost : kPairCost; }
// Positions of a step: one tile for each of a workgroup's four waves.
inline uint64_t attend_step(int format, int head_dim) {
  if (!four_bits(format)) return 128;
  return 4 * (head_dim == 64 ? kAttend4Tile<64> : head_dim == 128 ? kAttend4Tile<128> : kAttend4Tile<256>);
}

}  // namespace hllm_rocm
