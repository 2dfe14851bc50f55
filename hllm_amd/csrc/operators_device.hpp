// Device code that the operators' kernels share: vectors of eight values, the matrix product, copies into LDS and
// attention's cut of a batch's work into equal shares.
#pragma once

#include <atomic>
#include <climits>

#include "operators.hpp"

namespace hllm_rocm {
namespace {

constexpr int kThreads = 256;

typedef __bf16 bhalf;
typedef bhalf bhalf4 __attribute__((ext_vector_type(4)));
typedef bhalf bhalf8 __attribute__((ext_vector_type(8)));
typedef uint32_t uint2v __attribute__((ext_vector_type(2)));
typedef uint32_t uint4v __attribute__((ext_vector_type(4)));
typedef _Float16 half2v __attribute__((ext_vector_type(2)));

// ---------------------------------------------------------------- eight values

__device__ inline void load8(const _Float16* p, float* x) {
  const half8 h = *reinterpret_cast<const half8*>(p);
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = (float)h[i];
}
__device__ inline void load8(const bhalf* p, float* x) {
  const bhalf8 h = *reinterpret_cast<const bhalf8*>(p);
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = (float)h[i];
}
__device__ inline void load8(const float* p, float* x) {
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const floatx4 h = *reinterpret_cast<const floatx4*>(p + 4 * j);
#pragma unroll
    for (int i = 0; i < 4; ++i) x[4 * j + i] = h[i];
  }
}
__device__ inline void store8(_Float16* p, const float* x) {
  half8 h;
#pragma unroll
  for (int i = 0; i < 8; ++i) h[i] = (_Float16)x[i];
  *reinterpret_cast<half8*>(p) = h;
}
__device__ inline void store4(_Float16* p, floatx4 x) {
  *reinterpret_cast<half4*>(p) = half4{(_Float16)x[0], (_Float16)x[1], (_Float16)x[2], (_Float16)x[3]};
}
__device__ inline void store4(bhalf* p, floatx4 x) {
  *reinterpret_cast<bhalf4*>(p) = bhalf4{(bhalf)x[0], (bhalf)x[1], (bhalf)x[2], (bhalf)x[3]};
}
__device__ inline void store4(float* p, floatx4 x) { *reinterpret_cast<floatx4*>(p) = x; }
__device__ inline void store8(bhalf* p, const float* x) {
  bhalf8 h;
#pragma unroll
  for (int i = 0; i < 8; ++i) h[i] = (bhalf)x[i];
  *reinterpret_cast<bhalf8*>(p) = h;
}
__device__ inline void store8(float* p, const float* x) {
#pragma unroll
  for (int j = 0; j < 2; ++j) *reinterpret_cast<floatx4*>(p + 4 * j) = floatx4{x[4 * j], x[4 * j + 1], x[4 * j + 2], x[4 * j + 3]};
}

template <typename T>
__device__ inline T* at(const Strided& s, int row, int head, int d) {
  return static_cast<T*>(s.data) + (uint64_t)row * s.row + (uint64_t)head * s.head + d;
}

// ---------------------------------------------------------------- codes

// The values of four codes, in F32.
template <int F>
__device__ inline floatx4 decode4(uint32_t w) {
  if constexpr (F == HLLM_KV_E4M3) {
    const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
    return floatx4{lo[0], lo[1], hi[0], hi[1]};
  } else {
    return floatx4{(float)(int8_t)w, (float)(int8_t)(w >> 8), (float)(int8_t)(w >> 16), (float)(int8_t)(w >> 24)};
  }
}

// INT4 codes, held as code + 8, of the low and of the high four bits of a byte in either half of a word, as F16: beside 0x64 they are
// the numbers 1024 + n and 1024 + 16 n.
__device__ inline half2v low_halves(uint32_t w) {
  return __builtin_bit_cast(half2v, (w & 0x000f000fu) | 0x64006400u) - half2v{(_Float16)1032.0f, (_Float16)1032.0f};
}
__device__ inline half2v high_halves(uint32_t w) {
  const half2v sixteenth = {(_Float16)0.0625f, (_Float16)0.0625f}, bias = {(_Float16)-72.0f, (_Float16)-72.0f};
  return __builtin_elementwise_fma(__builtin_bit_cast(half2v, (w & 0x00f000f0u) | 0x64006400u), sixteenth, bias);
}
// The values of eight codes, in F32 and in order.
template <int F>
__device__ inline void values8(uint32_t w, float* x) {
  if constexpr (F == kE2m1) {
    const auto a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 0), b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 1),
               c = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 2), d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 3);
    x[0] = a[0], x[1] = a[1], x[2] = b[0], x[3] = b[1], x[4] = c[0], x[5] = c[1], x[6] = d[0], x[7] = d[1];
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = (float)((int)(w >> (4 * i) & 15u) - 8);
  }
}
// A group's scale. E2M1: the byte is a power of two's exponent + 127, 0 is 2^-127 (below F32's normal range) and 255 NaN. INT4: the
// upper half of an F32 number, of which those that are not finite stand for NaN, so that a group that holds nothing
// usable says so and no other group of its vector does.
template <int F>
__device__ inline float scale_of(uint32_t held) {
  const uint32_t bits = F == kE2m1 ? max(held << 23, 0x00400000u) : held << 16;
  return __uint_as_float((bits & 0x7f800000u) == 0x7f800000u ? 0x7fc00000u : bits);
}

// ---------------------------------------------------------------- attention

// More than 64 KiB of LDS is asked for once on each device.
inline void ask_for_lds(const void* kernel, int bytes, std::atomic<uint64_t>& asked) {
  int device = 0;
  HIP_CHECK(hipGetDevice(&device));
  if (asked.load(std::memory_order_relaxed) >> (device & 63) & 1) return;
  HIP_CHECK(hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, bytes));
  asked.fetch_or(1ull << (device & 63), std::memory_order_relaxed);
}

__device__ inline floatx4 mfma(half8 a, half8 b, floatx4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}
__device__ inline float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }
// The largest of a value over the four lanes of a column (lanes 16 apart), with the row swaps
// of the vector unit: shuffles through LDS cost 0.1 us a tile more.
__device__ inline float column_max(float v) {
  const auto half = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = fmaxf(__uint_as_float(half[0]), __uint_as_float(half[1]));
  const auto row = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(row[0]), __uint_as_float(row[1]));
}
__device__ inline float column_sum(float v) {
  v += __shfl_xor(v, 16, 64);
  return v + __shfl_xor(v, 32, 64);
}

// The largest over a wave, all of whose lanes are here.
template <int O>
__device__ inline uint32_t row_max(uint32_t v) {
  return max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x120 + O, 0xf, 0xf, false));
}
__device__ inline uint32_t wave_max(uint32_t v) {
  const auto half = __builtin_amdgcn_permlane32_swap(v, v, false, false);
  v = max(half[0], half[1]);
  const auto row = __builtin_amdgcn_permlane16_swap(v, v, false, false);
  v = max(row[0], row[1]);
  return row_max<1>(row_max<2>(row_max<4>(row_max<8>(v))));
}

// Copies into LDS as lds_copy16, of cache lines that are not kept: a step reads a layer's cache once. With nt /
// without, us, BF16, 8 KV heads of 128, caches not read just before: 3 x 200000 positions 204 / 229 (the first 6.2 TB/s, the
// read probe 6.3), 64 rows to 8192 43.4 / 49.5, 64 rows of 200 to 1000 18.5 / 20.4; one cache of 67 MB read again and again
// 17.3 / 17.1. Groups of more than sixteen query heads read a KV head twice, and lose the second reading's hits where
// the cache is small: groups of 20 over 2 KV heads 17.2 / 16.1 at 17 MB, 30.6 / 29.7 at 50 MB, 112 / 115 at 317 MB.
__device__ inline void lds_stream16(const void* sbase, uint32_t voffset, uint32_t lds_byte_offset) {
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1 nt" ::"v"(voffset), "s"(sbase),
               "s"(lds_byte_offset)
               : "memory", "m0");
#pragma clang diagnostic pop
}
// ... with an address a lane; and of one word a lane.
__device__ inline void lds_stream16_at(const void* from, uint32_t lds_byte_offset) {
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
  asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off nt" ::"v"(from), "s"(lds_byte_offset)
               : "memory", "m0");
#pragma clang diagnostic pop
}
// ... of lines that another workgroup of the die reads as well.
__device__ inline void lds_copy16_at(const void* from, uint32_t lds_byte_offset) {
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
  asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(from), "s"(lds_byte_offset)
               : "memory", "m0");
#pragma clang diagnostic pop
}
__device__ inline void lds_stream4_at(const void* from, uint32_t lds_byte_offset) {
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
  asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dword %0, off nt" ::"v"(from), "s"(lds_byte_offset)
               : "memory", "m0");
#pragma clang diagnostic pop
}

// Sum over the wave's lanes up to this one; lanes from `count` on do not matter.
__device__ inline int wave_scan(int v, int lane, int count) {
  for (int o = 1; o < 64 && o < count; o <<= 1) {
    const int below = __shfl_up(v, o, 64);
    if (lane >= o) v += below;
  }
  return v;
}

// The pairs (a row, a KV head, sixteen of its query heads) lie on a line, each as long as its steps of kStep
// positions (one tile a wave) and kCost more for starting it, and the line is cut into equal
// shares: a workgroup may end one pair, take whole ones and begin another.
template <int kStep>
__device__ inline int steps_of(int length) {
  return (length + kStep - 1) / kStep;
}
template <int kStep, int kCost>
__device__ inline int pair_units(int length) {
  return length < 0 ? 0 : steps_of<kStep>(length) + kCost;
}

// Where vector v of a pair's part i lies in the workspace. A share has two parts at most: of a pair
// that began before it and of one that goes on after it; and those of each of a cluster's pairs.
__device__ inline uint64_t part_at(const AttendArgs& a, int first, int i, int member, int v) {
  return (uint64_t)((i == 0 ? 2 * first + 1 : 2 * (first + i)) * a.cluster + member) * min(a.group, 16) + v;
}

// A workgroup's share, units from .. to of the line, and the pair it is at. Without `shared` a workgroup takes one pair.
template <int kStep, int kCost>
struct Share {
  int row, kvg, start, from = 0, to, budget = INT_MAX, length, units;

  // The share's first pair; false where there is none. in_row: pairs of a row; me: which of the `blocks` shares.
  __device__ inline bool first_pair(const AttendArgs& a, int in_row, int me, int blocks, int lane) {
    if (a.shared) {
      const int chunk = (a.rows + 63) / 64, lanes = (a.rows + chunk - 1) / chunk;  // rows of a lane, at most 16
      int own = 0, own_length = 0;
      for (int i = 0; i < chunk; ++i) {
        const int r = lane * chunk + i;
        if (r < a.rows) {
          own_length = min(a.lengths[r], a.limit);
          own += pair_units<kStep, kCost>(own_length) * in_row;
        }
      }
      int sum = wave_scan(own, lane, lanes);
      const int total = __builtin_amdgcn_readlane(sum, lanes - 1);
      budget = (total + blocks - 1) / blocks;
      from = me * budget;
      to = min(from + budget, total);
      if (from >= to) return false;
      int at = __builtin_ctzll(__ballot(sum > from));
      row = at * chunk;
      start = __builtin_amdgcn_readlane(sum - own, at);
      if (chunk > 1) {
        own_length = min(a.lengths[min(row + lane, a.rows - 1)], a.limit);
        own = lane < chunk && row + lane < a.rows ? pair_units<kStep, kCost>(own_length) * in_row : 0;
        sum = start + wave_scan(own, lane, chunk);
        at = __builtin_ctzll(__ballot(sum > from));
        row += at;
        start = __builtin_amdgcn_readlane(sum - own, at);
      }
      length = __builtin_amdgcn_readlane(own_length, at);
      units = pair_units<kStep, kCost>(length);
      kvg = (from - start) / units;
      start += kvg * units;
    } else {
      row = me / in_row;
      kvg = me - row * in_row;
      start = 0;
      length = min(uniform_load(a.lengths + row), a.limit);
      to = units = pair_units<kStep, kCost>(length);
      if (units == 0) return false;
    }
    return true;
  }
  // The next pair of the share, if there is one: rows of negative lengths have none.
  __device__ inline bool next_pair(const AttendArgs& a, int in_row) {
    start += units;
    if (start >= to) return false;
    if (++kvg < in_row) return true;
    kvg = 0;
    do {
      length = min(uniform_load(a.lengths + ++row), a.limit);
      units = pair_units<kStep, kCost>(length);
    } while (units == 0);
    return true;
  }
};

}  // namespace
}  // namespace hllm_rocm
