// Operators on a caller's device memory: rotary positions, the 8-bit paged KV cache (written and
// read back), and one new token's attention over it. The C entry points are at the end.
#include "operators.hpp"

#include <algorithm>
#include <atomic>
#include <climits>
#include <cmath>
#include <type_traits>

#include "abi.hpp"

namespace hllm_rocm {
namespace {

constexpr int kThreads = 256;
constexpr double kLog2e = 1.4426950408889634;

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

// ---------------------------------------------------------------- 8-bit codes

template <int F>
constexpr float kPeak = F == HLLM_KV_E4M3 ? 448.0f : 127.0f;

// Codes of eight values times `inverse`, to nearest even. The products are at most the largest
// code (by one rounding of a product more, which rounds back to it).
template <int F>
__device__ inline uint2v encode8(const float* x, float inverse) {
  uint2v w;
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    if constexpr (F == HLLM_KV_E4M3) {
      int c = __builtin_amdgcn_cvt_pk_fp8_f32(x[4 * j] * inverse, x[4 * j + 1] * inverse, 0, false);
      w[j] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(x[4 * j + 2] * inverse, x[4 * j + 3] * inverse, c, true);
    } else {
      uint32_t c = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int v = (int)fminf(fmaxf(rintf(x[4 * j + i] * inverse), -127.0f), 127.0f);
        c |= (uint32_t)(v & 255) << (8 * i);
      }
      w[j] = c;
    }
  }
  return w;
}

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

// ---------------------------------------------------------------- rotary positions

// cos and sin of position x turns, `turns` a 64-bit binary fraction of a turn: the fraction of the
// product is its low 64 bits, of which the upper 32 are kept (2^-32 turn is 1.5e-9 radians). Reduced to
// the nearest quarter turn, |x| <= pi / 4, where the Taylor series to x^9 and x^8 are off by at
// most 2e-9 and 3e-8; with the roundings of x (three of 2^-24, 1.5e-7) and of the sums sine and cosine are
// right to 5e-7.
__device__ inline float2 turn(int32_t position, uint64_t turns) {
  const uint32_t lo = (uint32_t)turns, hi = (uint32_t)(turns >> 32), p = (uint32_t)position;
  const uint32_t angle = __umulhi(p, lo) + p * hi - (position < 0 ? lo : 0u);
  const uint32_t quarter = (angle + 0x20000000u) >> 30;
  const float x = (float)(int32_t)(angle - (quarter << 30)) * 1.4629180792671596e-9f;  // 2 pi / 2^32
  const float y = x * x;
  const float s = x * (1.0f + y * (-1.0f / 6 + y * (1.0f / 120 + y * (-1.0f / 5040 + y * (1.0f / 362880)))));
  const float c = 1.0f + y * (-0.5f + y * (1.0f / 24 + y * (-1.0f / 720 + y * (1.0f / 40320))));
  const float a = quarter & 1 ? s : c, b = quarter & 1 ? c : s;
  return float2{quarter == 1 || quarter == 2 ? -a : a, quarter & 2 ? -b : b};
}

// One workgroup takes up to heads_per_block heads of one row, 16 elements of a head a thread,
// after its first threads have put the row's cosines and sines into LDS: they are computed once
// for all heads of the block, and no table is read. In half layout with a rotary
// dimension of whole sixteens a thread holds both elements of its pairs (eight of either half);
// interleaved pairs lie beside each other; other half layouts exchange through LDS (kExchange). So
// every pair is read before it is written and a tensor can be rotated in place. Bound by memory (a copy of
// 4 GiB reaches 4.8 TB/s): 8192 rows of 40 heads of 128 take 41 us in BF16 and 63 in F32, 4.1 and 5.4
// TB/s; interleaved pairs 44 and 64. The exchange sends every element through LDS as a word, turned or
// not: 24 of the 128 rotated 50 and 80 us, 3.4 and 4.2 TB/s.
//
// F >= 0: q_out is written as above, k is rotated and k and v are quantised: a head's lanes
// share its largest value by shuffles, and no rotated key is rounded or written in between. 2011 rows of 20 and 4
// heads of 256: 12.7 us, 4.3 TB/s; 64 rows 4.1 us, one chain of loads, sines, the largest value and the stores.
template <typename T, int F, bool kExchange>
__global__ void __launch_bounds__(kThreads) rotate_kernel(RotateArgs a) {
  __shared__ float2 cs[128];
  __shared__ float xs[kExchange ? kThreads * 17 : 1];
  const int row = blockIdx.x, t = threadIdx.x;
  const int R = a.rotary, half = R / 2;
  // The slot, the position and the elements are loaded together; a padding row's go unused.
  const int slot = F >= 0 ? uniform_load(a.slots + row) : 0, position = R > 0 ? uniform_load(a.positions + row) : 0;
  const int in_block = t / a.lanes, u = t - in_block * a.lanes;
  const int head = blockIdx.y * a.heads_per_block + in_block;
  const bool active = in_block < a.heads_per_block && head < a.q_heads + a.k_heads + a.v_heads;
  const bool is_q = head < a.q_heads, is_v = head >= a.q_heads + a.k_heads;
  const int h = is_q ? head : is_v ? head - a.q_heads - a.k_heads : head - a.q_heads;
  // The lane's two eights: of the pairs' halves, or of the halves of the elements that are not paired over
  // halves (from `rest` on), so that a head's lanes read whole lines.
  const bool over_halves = !kExchange && !a.interleaved && !is_v, paired = over_halves && 16 * u < R;
  const int rest = over_halves ? R : 0, before = rest / 16;
  const int d0 = kExchange ? 16 * u : paired ? 8 * u : rest + 8 * (u - before);
  const int d1 = kExchange ? d0 + 8 : paired ? half + 8 * u : d0 + (16 * a.lanes - rest) / 2;
  float x[16];
  if (active) {
    const Strided& in = is_q ? a.q : is_v ? a.v : a.k;
    load8(at<const T>(in, row, h, d0), x);
    load8(at<const T>(in, row, h, d1), x + 8);
  }
  if (F >= 0 && (slot < 0 || (slot >> a.pages.page_shift) >= a.pages.pages)) return;
  if (t < half) {
    const float2 v = turn(position, a.turns[t]);
    cs[t] = float2{v.x * a.magnitude, v.y * a.magnitude};
  }
  if constexpr (kExchange) {
#pragma unroll
    for (int i = 0; i < 16; ++i) xs[t * 17 + i] = active ? x[i] : 0.0f;
  }
  __syncthreads();
  if (!active) return;
  if (!is_v) {
    if constexpr (kExchange) {
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int d = 16 * u + i;
        if (d >= R) continue;
        const bool first = d < half;
        const int other = first ? d + half : d - half;
        const float2 v = cs[first ? d : other];
        const float y = xs[(t - u + (other >> 4)) * 17 + (other & 15)];
        x[i] = first ? x[i] * v.x - y * v.y : x[i] * v.x + y * v.y;
      }
    } else if (paired) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float2 v = cs[8 * u + i];
        const float x0 = x[i], x1 = x[8 + i];
        x[i] = x0 * v.x - x1 * v.y;
        x[8 + i] = x1 * v.x + x0 * v.y;
      }
    } else if (a.interleaved) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int d = i < 4 ? d0 + 2 * i : d1 + 2 * (i - 4);
        if (d >= R) continue;
        const float2 v = cs[d / 2];
        const float x0 = x[2 * i], x1 = x[2 * i + 1];
        x[2 * i] = x0 * v.x - x1 * v.y;
        x[2 * i + 1] = x1 * v.x + x0 * v.y;
      }
    }
  }
  if (F < 0 || is_q) {
    const Strided& out = is_q ? a.q_out : a.k_out;
    store8(at<T>(out, row, h, d0), x);
    store8(at<T>(out, row, h, d1), x + 8);
    return;
  }
  if constexpr (F >= 0) {
    // The bits of magnitudes order as the magnitudes, infinities and NaN above all others.
    uint32_t most = 0;
#pragma unroll
    for (int i = 0; i < 16; ++i) most = max(most, __float_as_uint(x[i]) & 0x7fffffffu);
    for (int o = 1; o < a.lanes; o <<= 1) most = max(most, (uint32_t)__shfl_xor((int)most, o, 64));
    const bool finite = most < 0x7f800000u;
    const float largest = fmaxf(__uint_as_float(finite ? most : 0u), 0x1p-100f);
    const float inverse = kPeak<F> / largest;
    if (!finite) {
#pragma unroll
      for (int i = 0; i < 16; ++i) x[i] = 0.0f;
    }
    const Pages& c = a.pages;
    const int page = slot >> c.page_shift, offset = slot & ((1 << c.page_shift) - 1);
    uint8_t* to = (is_v ? c.values : c.keys) + (uint64_t)page * c.page_stride + (uint64_t)offset * c.token_stride +
                  (uint64_t)h * c.head_stride;
    *reinterpret_cast<uint2v*>(to + d0) = encode8<F>(x, inverse);
    *reinterpret_cast<uint2v*>(to + d1) = encode8<F>(x + 8, inverse);
    if (u == 0) {
      float* scales = is_v ? c.value_scales : c.key_scales;
      scales[(((uint64_t)page * c.kv_heads + h) << c.page_shift) + offset] = finite ? largest / kPeak<F> : NAN;
    }
  }
}

// ---------------------------------------------------------------- reading back

// A thread reads the codes of sixteen bytes of output of a key, and of the value beside it, and writes
// them: a wave's accesses are whole lines (with sixteen codes a thread F32 stores were 64 bytes a
// lane apart: 3.5 TB/s). Nothing but memory traffic: 30000 positions of 8 heads of 128 to F16 32.6 us,
// 5.7 TB/s; F32 5.2 to 6.1.
template <typename T, int F, int D>
__global__ void __launch_bounds__(kThreads) kv_read_kernel(ReadArgs a) {
  constexpr int kCodes = 16 / sizeof(T), L = D / kCodes;
  const Pages& c = a.pages;
  const uint32_t per_row = (uint32_t)c.kv_heads * L;
  const uint64_t unit = (uint64_t)blockIdx.x * kThreads + threadIdx.x;
  const uint64_t row = unit / per_row;
  if (row >= (uint64_t)a.rows) return;
  const int in_row = (int)(unit - row * per_row), h = in_row / L, d = in_row % L * kCodes;
  const int slot = a.slots[row];
  if (slot < 0 || (slot >> c.page_shift) >= c.pages) return;
  const int page = slot >> c.page_shift, offset = slot & ((1 << c.page_shift) - 1);
  const uint64_t from = (uint64_t)page * c.page_stride + (uint64_t)offset * c.token_stride + (uint64_t)h * c.head_stride + d;
  const uint64_t scale_at = (((uint64_t)page * c.kv_heads + h) << c.page_shift) + offset;
  uint32_t codes[2][kCodes / 4];
#pragma unroll
  for (int j = 0; j < kCodes / 4; ++j) {
    codes[0][j] = reinterpret_cast<const uint32_t*>(c.keys + from)[j];
    codes[1][j] = reinterpret_cast<const uint32_t*>(c.values + from)[j];
  }
  const float scale[2] = {c.key_scales[scale_at], c.value_scales[scale_at]};
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    T* to = at<T>(which ? a.v : a.k, (int)row, h, d);
    if constexpr (kCodes == 8) {
      float x[8];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const floatx4 v = decode4<F>(codes[which][j]) * scale[which];
#pragma unroll
        for (int i = 0; i < 4; ++i) x[4 * j + i] = v[i];
      }
      store8(to, x);
    } else {
      store4(to, decode4<F>(codes[which][0]) * scale[which]);
    }
  }
}

// ---------------------------------------------------------------- attention

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

// Four codes as F16, which holds every code of either format exactly. INT8: with the sign bit
// turned over, the byte below 0x64 is the F16 number 1024 + 128 + code.
template <int F>
__device__ inline void halves4(uint32_t w, half2v& lo, half2v& hi) {
  if constexpr (F == HLLM_KV_E4M3) {
    lo = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, false);
    hi = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, true);
  } else {
    const half2v bias = {(_Float16)1152.0f, (_Float16)1152.0f};
    w ^= 0x80808080u;
    lo = __builtin_bit_cast(half2v, __builtin_amdgcn_perm(0x64646464u, w, 0x04010400u)) - bias;
    hi = __builtin_bit_cast(half2v, __builtin_amdgcn_perm(0x64646464u, w, 0x04030402u)) - bias;
  }
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
__device__ inline void lds_stream4_at(const void* from, uint32_t lds_byte_offset) {
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
  asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dword %0, off nt" ::"v"(from), "s"(lds_byte_offset)
               : "memory", "m0");
#pragma clang diagnostic pop
}

// A wave's tile of 32 positions in LDS: key and value rows and the 64 scales. A row's sixteen-byte
// chunks are permuted (chunk k at k ^ swizzle) so that the eight rows whose chunks are read at once
// lie in different banks.
template <int D>
struct Tile {
  static constexpr int kScales = 64 * D, kBytes = kScales + 256, kBlock = kThreads / 64 * kBytes;
  // Rows of keys (which = 0) and values, 64-byte rows with both of eight positions together.
  static __device__ int row_at(int which, int row) {
    if constexpr (D == 64) return (row >> 3) * 1024 + which * 512 + ((row & 7) ^ ((row >> 3) & 1)) * 64;
    return which * 32 * D + row * D;
  }
  static __device__ int swizzle(int row) { return D == 64 ? row & 3 : (row & 3) + 4 * ((row >> 3) & 1); }
};

// Sum over the wave's lanes up to this one; lanes from `count` on do not matter.
__device__ inline int wave_scan(int v, int lane, int count) {
  for (int o = 1; o < 64 && o < count; o <<= 1) {
    const int below = __shfl_up(v, o, 64);
    if (lane >= o) v += below;
  }
  return v;
}

// The pairs (a row, a KV head, sixteen of its query heads) lie on a line, each as long as its steps of 128
// positions (one tile a wave) and kPairCost more for starting it, and the line is cut into equal
// shares: a workgroup may end one pair, take whole ones and begin another.
__device__ inline int steps_of(int length) { return (length + 127) / 128; }
__device__ inline int pair_units(int length) { return length < 0 ? 0 : steps_of(length) + kPairCost; }

// Where vector v of a pair's part i lies in the workspace. A workgroup writes two parts at most: of a pair
// that began before it and of one that goes on after it.
__device__ inline uint64_t part_at(const AttendArgs& a, int first, int i, int v) {
  return (uint64_t)(i == 0 ? 2 * first + 1 : 2 * (first + i)) * min(a.group, 16) + v;
}

// A pair's scores S = K Q^T (positions x query heads) and sums O^T = V^T P are products on the matrix
// units: 16 query heads fill the columns of a 16 x 16 x 32 tile, so that groups of 1 to 16 heads read
// each position once and cost the same. Codes are exact in F16; a key's scale enters its score and a
// value's scale its weight, so no element is multiplied by a scale. The softmax (base 2) keeps its running
// maximum and sum in F32 and the tile's weights go from the score product to the value product in
// registers: with position 8 q + 4 h + i in row 4 q + i of score fragment h, a lane's scores are its
// operand of the value product.
//
// Bound by the cache's bytes where it is long: 6.1 TB/s at 3 x 200000 positions (a streaming read 6.3). A
// wave copies its next tile of 32 positions straight into LDS while it works on the last one, which is in registers by
// then: one tile a wave, so that 3 workgroups (D = 128) fit a CU. Two tiles a wave and half the workgroups took
// 31 us where this takes 26 (3 rows of 12000 to 30000 positions), tiles through registers 30. At
// some hundred positions a row it is bound by the chain of a workgroup's start (length, page numbers, first tile:
// 2.7 us) and the last round's imbalance: 64 rows to 2048 positions, 66 MB, 18.9 us. F32 tensors take twice
// as many products and LDS for twice the queries: 64 rows to 8192 33, 48, 99 us with the join at head dimensions 64, 128,
// 256, where BF16 takes 29, 43, 76.
template <typename T, int F, int D>
__global__ void __launch_bounds__(kThreads, kAttendBlocks<D>) kv_attention_kernel(AttendArgs a) {
  using Layout = Tile<D>;
  constexpr int KK = D / 32;   // 32-wide chunks of the score contraction
  constexpr int DF = D / 16;   // 16-row fragments of the output; a lane's value bytes of a position
  constexpr int VW = DF / 4;   // ... in words
  constexpr int P = sizeof(T) == 4 ? 2 : 1;  // F16 parts of a query element and of a weight
  extern __shared__ __attribute__((aligned(256))) char smem[];
  __shared__ float states[4][3][16];
  __shared__ half8 queries[P][KK][64];

  const Pages& c = a.pages;
  const int KVH = c.kv_heads, shift = c.page_shift, in_row = KVH * a.head_groups;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int quad = lane >> 4, col = lane & 15;
  const int me = blockIdx.x;
  const auto length_of = [&](int row) { return min(uniform_load(a.lengths + row), a.limit); };

  // The share, units from .. to of the line, and its first pair. Without `shared` a workgroup
  // takes one pair.
  int row, kvg, start, from = 0, to, budget = INT_MAX, length, units;
  if (a.shared) {
    const int chunk = (a.rows + 63) / 64, lanes = (a.rows + chunk - 1) / chunk;  // rows of a lane, at most 16
    int own = 0, own_length = 0;
    for (int i = 0; i < chunk; ++i) {
      const int r = lane * chunk + i;
      if (r < a.rows) {
        own_length = min(a.lengths[r], a.limit);
        own += pair_units(own_length) * in_row;
      }
    }
    int sum = wave_scan(own, lane, lanes);
    const int total = __builtin_amdgcn_readlane(sum, lanes - 1);
    budget = (total + (int)gridDim.x - 1) / (int)gridDim.x;
    from = me * budget;
    to = min(from + budget, total);
    if (from >= to) return;
    int at = __builtin_ctzll(__ballot(sum > from));
    row = at * chunk;
    start = __builtin_amdgcn_readlane(sum - own, at);
    if (chunk > 1) {
      own_length = min(a.lengths[min(row + lane, a.rows - 1)], a.limit);
      own = lane < chunk && row + lane < a.rows ? pair_units(own_length) * in_row : 0;
      sum = start + wave_scan(own, lane, chunk);
      at = __builtin_ctzll(__ballot(sum > from));
      row += at;
      start = __builtin_amdgcn_readlane(sum - own, at);
    }
    length = __builtin_amdgcn_readlane(own_length, at);
    units = pair_units(length);
    kvg = (from - start) / units;
    start += kvg * units;
  } else {
    row = me / in_row;
    kvg = me - row * in_row;
    start = 0;
    length = length_of(row);
    to = units = pair_units(length);
    if (units == 0) return;
  }
  // The next pair of the share, if there is one: rows of negative lengths have none.
  const auto next_pair = [&] {
    start += units;
    if (start >= to) return false;
    if (++kvg < in_row) return true;
    kvg = 0;
    do {
      length = length_of(++row);
      units = pair_units(length);
    } while (units == 0);
    return true;
  };

  bool again = false;
  for (bool more = true; more; more = next_pair()) {
  // This share's steps of the pair, low .. high - 1, and the workgroups that have others.
  const int steps = steps_of(length), first_unit = start + kPairCost;
  const int low = max(from - first_unit, 0), high = min(steps, to - first_unit);
  if (steps > 0 ? low >= high : start < from) continue;  // only the cost of starting it is this share's
  const int first = first_unit / budget;
  const int parts = a.shared && steps > 0 ? (first_unit + steps - 1) / budget - first + 1 : 1;
  const int kvh = kvg / a.head_groups, g0 = (kvg - kvh * a.head_groups) * 16;
  const int begin = 128 * low, end = min(length, 128 * high);
  if (again) __syncthreads();  // the workgroup has read the last pair's sums
  again = true;
  const int vectors = min(16, a.group - g0);

  const int32_t* table = a.table + (uint64_t)row * a.table_stride;
  const int mask = (1 << shift) - 1;
  const uint32_t token = c.token_stride;
  const uint8_t* keys = c.keys + (uint64_t)kvh * c.head_stride;
  const uint8_t* values = c.values + (uint64_t)kvh * c.head_stride;
  char* tile = smem + wave * Layout::kBytes;
  const uint32_t tile_at = (uint32_t)(size_t)((__attribute__((address_space(3))) char*)smem) + wave * Layout::kBytes;

  // One copy instruction takes 1 KiB, sixteen bytes a lane, all of one group of eight positions, which lies
  // in one page: the group's keys and values (D = 64), its keys (128) or half of them (256). The
  // chunks' order differs between even and odd groups.
  uint32_t lane_at[2];
  const uint8_t* lane_from[2];
#pragma unroll
  for (int odd = 0; odd < 2; ++odd) {
    constexpr int kChunks = D / 16;
    if constexpr (D == 64) {
      const int r = ((lane >> 2) & 7) ^ odd, chunk = (lane & 3) ^ Layout::swizzle(r);
      lane_from[odd] = (lane < 32 ? keys : values) + (uint32_t)r * token + chunk * 16;
    } else {
      const int r = lane / kChunks, chunk = lane % kChunks ^ Layout::swizzle(r + 8 * odd);
      lane_at[odd] = (uint32_t)r * token + chunk * 16;
    }
  }
  const float* lane_scales = lane < 32 ? c.key_scales : c.value_scales;
  // The table's entries of a tile's four groups (of the last position's group behind the part).
  int ids[4];
  const auto load_ids = [&](int t) {
#pragma unroll
    for (int g = 0; g < 4; ++g) ids[g] = uniform_load(table + (min(t + 8 * g, end - 1) >> shift));
  };
  // Starts a tile's copies; returns a bit for each group whose page is not there.
  const auto copy_tile = [&](int t) {
    int missing = 0, pages[4];
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const bool there = ids[g] >= 0 && ids[g] < c.pages;
      missing |= there ? 0 : 1 << g;
      pages[g] = there ? ids[g] : 0;
      const uint64_t page_at = (uint64_t)(uint32_t)pages[g] * c.page_stride + (uint64_t)(uint32_t)((t + 8 * g) & mask) * token;
      if constexpr (D == 64) {
        lds_stream16_at(lane_from[g & 1] + page_at, tile_at + g * 1024);
      } else {
#pragma unroll
        for (int i = 0; i < D / 128; ++i) {
          lds_stream16(keys + page_at + (uint64_t)(4 * i) * token, lane_at[g & 1], tile_at + (g * (D / 128) + i) * 1024);
          lds_stream16(values + page_at + (uint64_t)(4 * i) * token, lane_at[g & 1], tile_at + 32 * D + (g * (D / 128) + i) * 1024);
        }
      }
    }
    const int group = (lane & 31) >> 3;
    const int page = group & 2 ? (group & 1 ? pages[3] : pages[2]) : (group & 1 ? pages[1] : pages[0]);
    lds_stream4_at(lane_scales + ((((uint64_t)page * KVH + kvh) << shift) + ((t + (lane & 31)) & mask)), tile_at + Layout::kScales);
    return missing;
  };

  int t = begin + 32 * wave, missing = 0;
  if (t < end) {
    load_ids(t);
    missing = copy_tile(t);
    load_ids(min(t + 128, end - 1));
  }

  // Q^T as the B operand, kept in LDS for the four waves: chunk kk = 2 hh + s holds elements 64 hh + 16 quad + 8 s + j, the order
  // of a key's sixteen bytes. Each vector is divided by the power of two of its
  // largest element, which puts F32 and BF16 ranges into F16's and goes back into its scores.
  float factor, factor_lo;
  {
    float x[KK][8];
    const T* src = at<const T>(a.q, row, kvh * a.group + g0 + min(col, vectors - 1), 16 * quad);
    uint32_t most = 0;
#pragma unroll
    for (int kk = 0; kk < KK; ++kk) {
      load8(src + 64 * (kk >> 1) + 8 * (kk & 1), x[kk]);
#pragma unroll
      for (int j = 0; j < 8; ++j) most = max(most, __float_as_uint(x[kk][j]) & 0x7fffffffu);
    }
    most = max(most, (uint32_t)__shfl_xor((int)most, 16, 64));
    most = max(most, (uint32_t)__shfl_xor((int)most, 32, 64));
    // 2^e <= largest < 2^(e+1), e at most 126 (the largest numbers are left below 4); vectors that are
    // zero, below the normal range or not finite as they are.
    const uint32_t exponent = min(most >> 23, 253u);
    const bool usual = exponent >= 1 && most < 0x7f800000u;
    const float down = usual ? __uint_as_float((254u - exponent) << 23) : 1.0f;
    const float up = usual ? __uint_as_float(exponent << 23) : 1.0f;
    factor = a.scale_hi * up;
    factor_lo = a.scale_lo * up;
    if (wave == 0) {
#pragma unroll
      for (int kk = 0; kk < KK; ++kk) {
        half8 part[P];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float y = x[kk][j] * down;
          part[0][j] = (_Float16)y;
          if constexpr (P == 2) part[1][j] = (_Float16)(y - (float)part[0][j]);
        }
#pragma unroll
        for (int p = 0; p < P; ++p) queries[p][kk][lane] = part[p];
      }
    }
  }
  __syncthreads();

  // The weights of a position are 2^(score - m) times its value scale; they enter the products
  // divided by r, and so do the sums o. r is a weight that was the largest once: it follows m, and is
  // raised when a weight is 2^12 times as large, so that o is seldom rescaled and F16 holds
  // every weight to 2^-11 or to 2^-25 of the largest. One F16 part for 16-bit tensors, whose outputs are
  // rounded as coarsely: 64 rows to 2048 in F16 are off by 2.4e-4 against 2.1e-4 for the plain form with F32 weights; two parts
  // took 23.3 -> 24.0 us there, 58.2 -> 59.8 for 256 rows, 30.0 -> 30.5 for 3 long ones.
  floatx4 o[DF];
#pragma unroll
  for (int f = 0; f < DF; ++f) o[f] = floatx4{0.f, 0.f, 0.f, 0.f};
  float m = -INFINITY, l = 0.0f, r = 0.0f;
  bool any = false;  // whether the wave has had a position

  // Score fragment h's row 4 q + i is position 8 q + 4 h + i: a lane's scores are the eight
  // positions 8 quad .. + 7, which are also its slots of the value products.
  const int key_row = 8 * (col >> 2) + (col & 3);
  const int key_lane = Layout::row_at(0, key_row) + ((quad ^ Layout::swizzle(key_row)) * 16);
  const int value_lane = Layout::row_at(1, 8 * quad) + ((DF * col / 16 ^ Layout::swizzle(8 * quad)) * 16) + DF * col % 16;
  for (; t < end; t += 128) {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    const int gone = missing;
    const bool whole = gone == 0 && t + 32 <= end;
    any |= gone != 15;  // groups behind the end count as the last one's page
    if (!whole) {
      // Values of positions past the part and in pages that are not there, whatever they are.
      const int own = lane >> 1;
      if (t + own >= end || (gone >> (own >> 3)) & 1) {
        char* line = tile + Layout::row_at(1, own) + (lane & 1) * (D / 2);
#pragma unroll
        for (int i = 0; i < D / 32; ++i) *reinterpret_cast<uint4v*>(line + 16 * i) = uint4v{0, 0, 0, 0};
        reinterpret_cast<float*>(tile + Layout::kScales)[32 + own] = 0.0f;
      }
    }
    floatx4 s0 = {0.f, 0.f, 0.f, 0.f}, s1 = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int hh = 0; hh < D / 64; ++hh) {
      const int at_hh = (key_lane ^ (hh & 1) * 64) + (hh >> 1) * 128;
      uint4v kw[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) kw[h] = *reinterpret_cast<const uint4v*>(tile + at_hh + 4 * D * h);
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        half8 k[2];
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int w = 0; w < 2; ++w) {
            half2v lo, hi;
            halves4<F>(kw[h][2 * s + w], lo, hi);
            k[h][4 * w] = lo[0];
            k[h][4 * w + 1] = lo[1];
            k[h][4 * w + 2] = hi[0];
            k[h][4 * w + 3] = hi[1];
          }
#pragma unroll
        for (int p = 0; p < P; ++p) {
          const half8 q = queries[p][2 * hh + s][lane];
          s0 = mfma(k[0], q, s0);
          s1 = mfma(k[1], q, s1);
        }
      }
    }
    // F32 tensors keep the scores' factors as sums of two floats and round a score once, after the
    // maximum is taken away: a score of some tens rounded by itself moves its weight by 1e-6.
    float sc[8], ks[8], by_lo[8], vs[8];
    load8(reinterpret_cast<const float*>(tile + Layout::kScales) + 8 * quad, ks);
    load8(reinterpret_cast<const float*>(tile + Layout::kScales) + 32 + 8 * quad, vs);
    uint32_t vw[8][VW];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const char* line = D == 64 ? tile + (value_lane ^ (j * 64 + (j & 3) * 16)) : tile + (value_lane ^ (j & 3) * 16) + j * D;
      if constexpr (VW == 1) vw[j][0] = *reinterpret_cast<const uint32_t*>(line);
      if constexpr (VW == 2) {
        const uint2v w = *reinterpret_cast<const uint2v*>(line);
        vw[j][0] = w[0];
        vw[j][1] = w[1];
      }
      if constexpr (VW == 4) {
        const uint4v w = *reinterpret_cast<const uint4v*>(line);
#pragma unroll
        for (int i = 0; i < 4; ++i) vw[j][i] = w[i];
      }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float d = i < 4 ? s0[i & 3] : s1[i & 3];
      const float by = ks[i] * factor;
      sc[i] = d * by;
      if constexpr (P == 2)
        by_lo[i] = sc[i] == -INFINITY ? 0.0f : fmaf(d, by, -sc[i]) + d * (fmaf(ks[i], factor, -by) + ks[i] * factor_lo);
    }
    if (!whole) {
      const int valid = (gone >> quad) & 1 ? 0 : end - (t + 8 * quad);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        sc[i] = i < valid ? sc[i] : -INFINITY;
        if constexpr (P == 2) by_lo[i] = i < valid ? by_lo[i] : 0.0f;
      }
    }
    // The tile is in registers: the next one's copies start.
    if (t + 128 < end) {
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      missing = copy_tile(t + 128);
      load_ids(min(t + 256, end - 1));
    }
    float most = sc[0];
#pragma unroll
    for (int i = 1; i < 8; ++i) most = fmaxf(most, sc[i]);
    const float m_new = fmaxf(m, column_max(most));
    const float base = m_new == -INFINITY ? 0.0f : m_new;
    const float decay = exp2_fast(m - base);
    float weight[8], sum = 0.0f, largest = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float p = exp2_fast(P == 2 ? (sc[i] - base) + by_lo[i] : sc[i] - base);
      sum += p;
      weight[i] = p * vs[i];
      largest = fmaxf(largest, fabsf(weight[i]));  // a caller's own scales may be negative
    }
    l = l * decay + sum;
    m = m_new;
    r *= decay;
    largest = column_max(largest);
    if (__any(largest > 4096.0f * r)) {
      const float raised = fmaxf(r, largest), rescale = raised > r ? r / raised : 1.0f;
#pragma unroll
      for (int f = 0; f < DF; ++f) o[f] *= rescale;
      r = raised;
    }
    const float over = r > 0x1p-125f ? __builtin_amdgcn_rcpf(r) : 0.0f;  // smaller weights are nothing
    half8 pf[P];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      float w = weight[i] * over;
      // As a value of its own: rounded with the product in one step, the first part would differ
      // from the one that the second part is the rest of.
      if constexpr (P == 2) asm("" : "+v"(w));
      pf[0][i] = (_Float16)w;
      if constexpr (P == 2) pf[1][i] = (_Float16)(w - (float)pf[0][i]);
    }
    // Value words w: bytes 4 w .. + 3 of eight positions; two positions' bytes are paired, then
    // widened. Fragment f's row c is element DF c + f.
#pragma unroll
    for (int w = 0; w < VW; ++w) {
      half8 v[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t lo = __builtin_amdgcn_perm(vw[2 * j + 1][w], vw[2 * j][w], 0x05010400u);
        const uint32_t hi = __builtin_amdgcn_perm(vw[2 * j + 1][w], vw[2 * j][w], 0x07030602u);
        half2v x[4];
        halves4<F>(lo, x[0], x[1]);
        halves4<F>(hi, x[2], x[3]);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          v[i][2 * j] = x[i][0];
          v[i][2 * j + 1] = x[i][1];
        }
      }
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int p = 0; p < P; ++p) o[4 * w + i] = mfma(v[i], pf[p], o[4 * w + i]);
    }
  }

  // The four waves' states meet in LDS, each wave's in its own tile.
  l = column_sum(l);
  // Only scores of -inf (an infinite query's): a sum that is not 0 beside that maximum tells them from no positions.
  if (any && l == 0.0f) l = 1.0f;
  if (quad == 0) {
    states[wave][0][col] = m;
    states[wave][1][col] = l;
    states[wave][2][col] = r;
  }
  static_assert(Layout::kBytes >= 4 * DF * 64 * 4, "a wave's sums lie in its tile");
  // A lane's component i of four fragments: four elements that follow one another.
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int k = 0; k < VW; ++k)
      reinterpret_cast<floatx4*>(tile)[(i * VW + k) * 64 + lane] = floatx4{o[4 * k][i], o[4 * k + 1][i], o[4 * k + 2][i], o[4 * k + 3][i]};
  __syncthreads();
  T* out = at<T>(a.out, row, kvh * a.group + g0, 0);
  if (a.cuts && low == 0 && threadIdx.x == 0) a.cuts[row * in_row + kvg] = int2{first, parts};
  for (int e = threadIdx.x; e < vectors * (D / 4); e += kThreads) {
    const int v = e / (D / 4), d = e % (D / 4) * 4;
    float top = -INFINITY, total = 0.0f, held = 0.0f;
    floatx4 x[4];
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      x[w] = reinterpret_cast<const floatx4*>(smem + w * Layout::kBytes)[(d / DF % 4 * VW + d % DF / 4) * 64 + d / (4 * DF) * 16 + v];
      top = fmaxf(top, states[w][0][v]);
      held += states[w][1][v];
    }
    const float base = top == -INFINITY ? 0.0f : top;
    float decay[4];
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      decay[w] = exp2_fast(states[w][0][v] - base);
      total += states[w][1][v] * decay[w];
    }
    // Divided by the total before r's share of a value scale enters: a mean of large values is finite, their sum may not be.
    const float inverse = total == 0.0f ? 0.0f : 1.0f / total;
    floatx4 y = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < 4; ++w) y += x[w] * inverse * (states[w][2][v] * decay[w]);
    const bool undefined = total == 0.0f && held != 0.0f;  // no softmax of scores that are all -inf
    if (parts == 1) {
      store4(out + v * a.out.head + d, undefined ? floatx4{NAN, NAN, NAN, NAN} : y);
    } else {
      if (undefined) total = 1.0f;  // NaN in the join, unless another part has finite scores
      const uint64_t part = part_at(a, first, me - first, v);
      *reinterpret_cast<floatx4*>(a.part + part * D + d) = y;
      if (d == 0) *reinterpret_cast<float2*>(a.stats + 2 * part) = float2{top, total};
    }
  }
  }
}

__device__ inline float first_lane(float v) { return __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(v))); }
__device__ inline int2 uniform_cut(const int2* p) {
  return int2{uniform_load(&p->x), uniform_load(&p->y)};
}

// Joins the parts of the pairs that were cut, one wave for a query head: each part's output weighted
// with its share of the softmax sum. A part's vector takes D / 4 lanes, so a wave reads up to four parts at
// once, and eight times as many before it uses them: the kernel is a few memory round trips long (64 rows
// of 32 heads 4.0 us, 3 rows of up to 30 parts a pair 4.9). A workgroup that joined the parts itself when it was the last
// to arrive took 3 to 8 us longer: its stores and counts have to reach the other dies' caches.
template <typename T, int D>
__global__ void __launch_bounds__(kThreads) kv_join_kernel(AttendArgs a) {
  constexpr int kLanes = D / 4, kSlots = 64 / kLanes, kDeep = 8;
  const int vector = blockIdx.x * (kThreads / 64) + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  if (vector >= a.rows * a.q_heads) return;
  const int row = vector / a.q_heads, head = vector - row * a.q_heads, kvh = head / a.group, g = head - kvh * a.group;
  const int length = uniform_load(a.lengths + row);
  const int2 cut = uniform_cut(a.cuts + (row * a.pages.kv_heads + kvh) * a.head_groups + g / 16);
  const int first = cut.x, parts = cut.y;
  if (min(length, a.limit) <= 0 || parts <= 1) return;  // a row without positions has no cut there
  const int v = g % 16, slot = lane / kLanes, d = lane % kLanes * 4;
  const auto stat = [&](int i) { return *reinterpret_cast<const float2*>(a.stats + 2 * part_at(a, first, min(i, parts - 1), v)); };
  floatx4 y = {0.f, 0.f, 0.f, 0.f};
  float top = -INFINITY, total = 0.0f;
  bool held = false;
  for (int i0 = 0; i0 < parts; i0 += 64) {
    // Statistics and the first outputs of 64 parts are loaded together.
    const int n = min(64, parts - i0);
    const float2 own = stat(i0 + lane);
    float most = lane < n ? own.x : -INFINITY, weight = 0.0f;
    for (int j0 = 0; j0 < n; j0 += kSlots * kDeep) {
      floatx4 x[kDeep];
#pragma unroll
      for (int j = 0; j < kDeep; ++j)
        x[j] = *reinterpret_cast<const floatx4*>(a.part + part_at(a, first, i0 + min(j0 + j * kSlots + slot, n - 1), v) * D + d);
      if (j0 == 0) {
        // The first lanes hold the parts: as many steps as those take, and the result from lane 0.
        for (int o = 1; o < n; o <<= 1) most = fmaxf(most, __shfl_xor(most, o, 64));
        most = fmaxf(first_lane(most), top);
        // A part holds nothing where its sum is 0. The maximum does not tell: NaN scores leave it at -inf and
        // the sum NaN, which goes on to the output.
        const float base = most == -INFINITY ? 0.0f : most, before = total * exp2_fast(top - base);
        top = most;
        weight = lane < n ? exp2_fast(own.x - base) * own.y : 0.0f;
        held |= __any(lane < n && own.y != 0.0f);
        // y is kept divided by the total: means of large values are finite, their sums may not be.
        total = weight;
        for (int o = 1; o < n; o <<= 1) total += __shfl_xor(total, o, 64);
        total = first_lane(total) + before;
        const float inverse = total == 0.0f ? 0.0f : 1.0f / total;
        weight *= inverse;
        y *= before * inverse;
      }
#pragma unroll
      for (int j = 0; j < kDeep; ++j) {
        const int i = j0 + j * kSlots + slot;
        const float w = __shfl(weight, min(i, 63), 64);
        if (i < n) y += x[j] * w;
      }
    }
  }
  for (int o = kLanes; o < 64; o <<= 1) {
#pragma unroll
    for (int i = 0; i < 4; ++i) y[i] += __shfl_xor(y[i], o, 64);
  }
  const bool undefined = total == 0.0f && held;  // no softmax of scores that are all -inf
  if (slot == 0) store4(at<T>(a.out, row, head, d), undefined ? floatx4{NAN, NAN, NAN, NAN} : y);
}

// Threads for a row's heads of `lanes` lanes in one workgroup of rotate_kernel, and its workgroups.
int rotate_threads(const RotateArgs& a) { return std::min(kThreads, ((a.q_heads + a.k_heads + a.v_heads) * a.lanes + 63) / 64 * 64); }
int rotate_blocks(const RotateArgs& a) {
  const int heads = a.q_heads + a.k_heads + a.v_heads, per_block = rotate_threads(a) / a.lanes;
  return (heads + per_block - 1) / per_block;
}

template <typename T, int F>
void rotate(hipStream_t stream, int rows, const RotateArgs& a) {
  const int threads = rotate_threads(a);
  RotateArgs b = a;
  b.heads_per_block = threads / a.lanes;
  const dim3 grid(rows, rotate_blocks(a));
  // The block's first rotary / 2 threads compute the cosines.
  const int block = std::max(threads, (a.rotary / 2 + 63) / 64 * 64);
  if (!a.interleaved && a.rotary % 16)
    rotate_kernel<T, F, true><<<grid, block, 0, stream>>>(b);
  else
    rotate_kernel<T, F, false><<<grid, block, 0, stream>>>(b);
}

template <typename T>
void rotate_to(hipStream_t stream, int format, int rows, const RotateArgs& a) {
  if (format < 0) return rotate<T, -1>(stream, rows, a);
  if (format == HLLM_KV_E4M3) return rotate<T, HLLM_KV_E4M3>(stream, rows, a);
  rotate<T, HLLM_KV_INT8>(stream, rows, a);
}

template <typename T, int F>
void kv_read(hipStream_t stream, int head_dim, const ReadArgs& a) {
  const uint64_t units = (uint64_t)a.rows * a.pages.kv_heads * (head_dim * sizeof(T) / 16);
  const unsigned blocks = (unsigned)((units + kThreads - 1) / kThreads);
  if (head_dim == 64) kv_read_kernel<T, F, 64><<<blocks, kThreads, 0, stream>>>(a);
  if (head_dim == 128) kv_read_kernel<T, F, 128><<<blocks, kThreads, 0, stream>>>(a);
  if (head_dim == 256) kv_read_kernel<T, F, 256><<<blocks, kThreads, 0, stream>>>(a);
}

template <typename T, int F, int D>
void attend(hipStream_t stream, const AttendArgs& a) {
  constexpr int kLds = Tile<D>::kBlock;
  // More than 64 KiB of LDS is asked for once on each device.
  static std::atomic<uint64_t> asked{0};
  int device = 0;
  HIP_CHECK(hipGetDevice(&device));
  if (!(asked.load(std::memory_order_relaxed) >> (device & 63) & 1)) {
    HIP_CHECK(hipFuncSetAttribute(reinterpret_cast<const void*>(&kv_attention_kernel<T, F, D>),
                                  hipFuncAttributeMaxDynamicSharedMemorySize, kLds));
    asked.fetch_or(1ull << (device & 63), std::memory_order_relaxed);
  }
  kv_attention_kernel<T, F, D><<<a.blocks, kThreads, kLds, stream>>>(a);
  if (a.cuts) kv_join_kernel<T, D><<<(unsigned)(a.rows * a.q_heads + 3) / 4, kThreads, 0, stream>>>(a);
}
template <typename T, int F>
void attend_dim(hipStream_t stream, int head_dim, const AttendArgs& a) {
  if (head_dim == 64) attend<T, F, 64>(stream, a);
  if (head_dim == 128) attend<T, F, 128>(stream, a);
  if (head_dim == 256) attend<T, F, 256>(stream, a);
}

template <typename T>
void attend_format(hipStream_t stream, int format, int head_dim, const AttendArgs& a) {
  if (format == HLLM_KV_E4M3) return attend_dim<T, HLLM_KV_E4M3>(stream, head_dim, a);
  attend_dim<T, HLLM_KV_INT8>(stream, head_dim, a);
}

}  // namespace

void launch_rotate(hipStream_t stream, uint32_t dtype, int format, int rows, const RotateArgs& a) {
  if (dtype == HLLM_DTYPE_F16) return rotate_to<_Float16>(stream, format, rows, a);
  if (dtype == HLLM_DTYPE_BF16) return rotate_to<bhalf>(stream, format, rows, a);
  rotate_to<float>(stream, format, rows, a);
}

void launch_kv_read(hipStream_t stream, uint32_t dtype, int format, int head_dim, const ReadArgs& a) {
  const auto run = [&](auto zero) {
    using T = decltype(zero);
    if (format == HLLM_KV_E4M3)
      kv_read<T, HLLM_KV_E4M3>(stream, head_dim, a);
    else
      kv_read<T, HLLM_KV_INT8>(stream, head_dim, a);
  };
  if (dtype == HLLM_DTYPE_F16) return run(_Float16{});
  if (dtype == HLLM_DTYPE_BF16) return run(bhalf{});
  run(0.0f);
}

void launch_kv_attention(hipStream_t stream, uint32_t dtype, int format, int head_dim, const AttendArgs& a) {
  if (dtype == HLLM_DTYPE_F16) return attend_format<_Float16>(stream, format, head_dim, a);
  if (dtype == HLLM_DTYPE_BF16) return attend_format<bhalf>(stream, format, head_dim, a);
  attend_format<float>(stream, format, head_dim, a);
}

// ---------------------------------------------------------------- argument checks

namespace {

// Rows of one call, and workgroups of kThreads threads of one launch: below 2^32 threads over all of a grid's dimensions.
constexpr uint64_t kMostRows = 1u << 20;
constexpr uint64_t kMostBlocks = (1u << 24) - 1;

[[noreturn]] void refuse(const std::string& message) { fail(HLLM_INVALID_REQUEST, message); }

size_t element_size(uint32_t dtype) { return dtype == HLLM_DTYPE_F32 ? 4 : 2; }

// Whether vectors of `width` at strides a (of na) and b (of nb) are apart, one inside the other.
bool apart(uint64_t width, uint64_t na, uint64_t a, uint64_t nb, uint64_t b) {
  const auto nested = [&](uint64_t ni, uint64_t i, uint64_t no, uint64_t o) {
    uint64_t extent = width;
    if (ni > 1) {
      if (i < width) return false;
      extent = (ni - 1) * i + width;
    }
    return no <= 1 || o >= extent;
  };
  return nested(na, a, nb, b) || nested(nb, b, na, a);
}

Strided tensor(const hllm_rocm_tensor* t, const char* name, uint64_t rows, uint64_t width, bool output) {
  const std::string who = name;
  if (!t) refuse(who + " is null");
  if (!t->data) refuse(who + " has no memory");
  if (t->dtype != HLLM_DTYPE_F32 && t->dtype != HLLM_DTYPE_F16 && t->dtype != HLLM_DTYPE_BF16) refuse(who + ": unknown dtype");
  if (t->heads < 1 || t->heads > 1024) refuse(who + ": 1 to 1024 heads");
  const size_t size = element_size(t->dtype);
  if ((uintptr_t)t->data % 16) refuse(who + ": memory must be 16-byte aligned");
  if (t->row_stride > (1ull << 40) || t->head_stride > (1ull << 40)) refuse(who + ": stride too large");
  if ((rows > 1 && t->row_stride * size % 16) || (t->heads > 1 && t->head_stride * size % 16))
    refuse(who + ": strides must be multiples of 16 bytes");
  if (output && !apart(width, rows, t->row_stride, t->heads, t->head_stride)) refuse(who + ": its vectors overlap");
  return {t->data, t->row_stride, t->head_stride};
}

// An output that starts where its input does has to be that input.
void check_in_place(const hllm_rocm_tensor* in, const hllm_rocm_tensor* out, uint64_t rows) {
  if (in->data != out->data) return;
  if ((rows > 1 && in->row_stride != out->row_stride) || (in->heads > 1 && in->head_stride != out->head_stride))
    refuse("an output in its input's memory must have its strides");
}

// Two outputs, or an output and another tensor's input, that start at one address.
void check_apart(const void* a, const char* name_a, const void* b, const char* name_b) {
  if (a == b) refuse(std::string(name_a) + " and " + name_b + " are one memory");
}

void check_rows(uint64_t rows) {
  if (rows > kMostRows) refuse("at most 1048576 rows a call");
}

void check_rotate_grid(uint64_t rows, const RotateArgs& a) {
  if (rows * rotate_blocks(a) > kMostBlocks) refuse("too many rows for these heads");
}

Pages pages_of(const hllm_rocm_kv_pages* p) {
  if (!p) refuse("pages is null");
  if (p->format != HLLM_KV_E4M3 && p->format != HLLM_KV_INT8) refuse("unknown cache format");
  if (p->head_dimension != 64 && p->head_dimension != 128 && p->head_dimension != 256)
    refuse("a cache's head dimension is 64, 128 or 256");
  if (p->kv_heads < 1 || p->kv_heads > 1024) refuse("1 to 1024 key-value heads");
  if (p->page_tokens < 8 || p->page_tokens > 4096 || (p->page_tokens & (p->page_tokens - 1)))
    refuse("a page's tokens are a power of two, 8 to 4096");
  if (p->pages < 1 || (uint64_t)p->pages * p->page_tokens > 0x7fffffffull) refuse("a cache has 1 to 2^31 - 1 slots");
  if (!p->keys || !p->values || !p->key_scales || !p->value_scales) refuse("a cache's memory is null");
  if (((uintptr_t)p->keys | (uintptr_t)p->values | (uintptr_t)p->key_scales | (uintptr_t)p->value_scales) % 16)
    refuse("a cache's memory must be 16-byte aligned");
  if (p->page_stride >= (1ull << 32) || p->token_stride > (1ull << 28) || p->head_stride > (1ull << 40))
    refuse("a cache's stride is too large");
  if ((p->pages > 1 && p->page_stride % 16) || p->token_stride % 16 || (p->kv_heads > 1 && p->head_stride % 16))
    refuse("a cache's strides must be multiples of 16 bytes");
  const uint64_t head = p->kv_heads > 1 ? p->head_stride : 0;
  const uint64_t extent = (p->page_tokens - 1) * p->token_stride + (p->kv_heads - 1) * head + p->head_dimension;
  if (!apart(p->head_dimension, p->page_tokens, p->token_stride, p->kv_heads, head) ||
      (p->pages > 1 && p->page_stride < extent))
    refuse("a cache's vectors overlap");
  int shift = 0;
  while ((1u << shift) < p->page_tokens) ++shift;
  return {static_cast<uint8_t*>(p->keys), static_cast<uint8_t*>(p->values), p->key_scales, p->value_scales,
          p->pages > 1 ? (uint32_t)p->page_stride : 0u, (uint32_t)p->token_stride, head, (int32_t)p->pages, shift, (int32_t)p->kv_heads};
}

void check_rope(const hllm_rocm_rope* rope, uint64_t head_dim) {
  if (!rope) refuse("rope is null");
  if (rope->rotary_dimension < 2 || rope->rotary_dimension > 256 || rope->rotary_dimension % 2 ||
      rope->layout > HLLM_ROPE_INTERLEAVED)
    refuse("rope is no plan of hllm_rocm_rope_plan");
  if (rope->rotary_dimension > head_dim) refuse("the rotary dimension is larger than the head's");
}

void take_rope(const hllm_rocm_rope* rope, const int32_t* positions, RotateArgs& a) {
  if (!positions) refuse("positions is null");
  a.positions = positions;
  a.rotary = (int32_t)rope->rotary_dimension;
  a.interleaved = rope->layout == HLLM_ROPE_INTERLEAVED;
  a.magnitude = rope->magnitude;
  std::copy(rope->turns, rope->turns + 128, a.turns);
}

// The call's device for its scope.
class OnDevice {
 public:
  explicit OnDevice(int32_t device) {
    HIP_CHECK(hipGetDevice(&before_));
    if (before_ != device) {
      // Asked first: the error of a failed hipSetDevice would be reported by the next launch.
      int devices = 0;
      HIP_CHECK(hipGetDeviceCount(&devices));
      if (device >= devices) refuse("there is no device " + std::to_string(device));
      HIP_CHECK(hipSetDevice(device));
      changed_ = true;
    }
  }
  ~OnDevice() {
    if (changed_) (void)hipSetDevice(before_);
  }

 private:
  int before_ = 0;
  bool changed_ = false;
};

void check_device(int32_t device) {
  if (device < 0) refuse("device is negative");
}

double positive(double x, double standard, const char* name) {
  if (x == 0.0) x = standard;
  if (!(x > 0.0) || !std::isfinite(x)) refuse(std::string(name) + " must be positive");
  return x;
}

void plan_rope(const hllm_rocm_rope_config& c, hllm_rocm_rope& out) {
  const uint32_t n = c.rotary_dimension;
  if (n < 2 || n > 256 || n % 2) refuse("the rotary dimension is even, 2 to 256");
  if (c.layout > HLLM_ROPE_INTERLEAVED) refuse("unknown rope layout");
  if (c.scaling > HLLM_ROPE_YARN) refuse("unknown rope scaling");
  if (!(c.theta > 1.0) || !std::isfinite(c.theta)) refuse("theta must be greater than 1");
  const long double turn = 2 * 3.14159265358979323846264338327950288L;
  long double factor = 1, length = 0, low = 0, high = 0, first = 0, last = 0;
  hllm_rocm_rope r{};
  r.rotary_dimension = n;
  r.layout = c.layout;
  r.magnitude = 1.0f;
  if (c.scaling != HLLM_ROPE_UNSCALED) {
    if (!(c.factor >= 1.0) || !std::isfinite(c.factor)) refuse("factor must be at least 1");
    factor = c.factor;
  }
  if (c.scaling == HLLM_ROPE_LLAMA3 || c.scaling == HLLM_ROPE_YARN) length = positive(c.original_length, 0.0, "original_length");
  if (c.scaling == HLLM_ROPE_LLAMA3) {
    low = positive(c.low_frequency_factor, 0.0, "low_frequency_factor");
    high = positive(c.high_frequency_factor, 0.0, "high_frequency_factor");
    if (!(high > low)) refuse("high_frequency_factor must be greater than low_frequency_factor");
  }
  if (c.scaling == HLLM_ROPE_YARN) {
    const long double fast = positive(c.beta_fast, 32.0, "beta_fast"), slow = positive(c.beta_slow, 1.0, "beta_slow");
    if (!(fast > slow)) refuse("beta_fast must be greater than beta_slow");
    // The pair index that turns `turns` times over the original length.
    const auto pair = [&](long double turns) {
      return n * std::log(length / (turns * turn)) / (2 * std::log((long double)c.theta));
    };
    first = std::max(0.0L, std::floor(pair(fast)));
    last = std::min((long double)n - 1, std::ceil(pair(slow)));
    r.magnitude = (float)positive(c.magnitude, 0.1 * std::log(c.factor) + 1.0, "magnitude");
    if (!(r.magnitude > 0.0f) || !std::isfinite(r.magnitude)) refuse("magnitude is no F32 number");
  }
  const long double step = -2.0L * std::log((long double)c.theta) / n;
  for (uint32_t i = 0; i < n / 2; ++i) {
    long double f = std::exp(step * i);
    if (c.scaling == HLLM_ROPE_LINEAR) f /= factor;
    if (c.scaling == HLLM_ROPE_LLAMA3) {
      const long double keep = std::clamp((length * f / turn - low) / (high - low), 0.0L, 1.0L);
      f = f * keep + f / factor * (1 - keep);
    }
    if (c.scaling == HLLM_ROPE_YARN) {
      const long double ramp = std::clamp((i - first) / std::max(0.001L, last - first), 0.0L, 1.0L);
      f = f * (1 - ramp) + f / factor * ramp;
    }
    r.turns[i] = (uint64_t)std::llround(std::ldexp(f / turn, 64));  // f <= 1: below 2^62
  }
  out = r;
}

}  // namespace
}  // namespace hllm_rocm

// ========================================================================= C ABI

using namespace hllm_rocm;

extern "C" {

hllm_status hllm_rocm_rope_plan(const hllm_rocm_rope_config* config, hllm_rocm_rope* out) {
  return guarded([&] {
    if (!config || !out) refuse("null argument");
    plan_rope(*config, *out);
  });
}

hllm_status hllm_rocm_rope_apply(int32_t device, void* stream, const hllm_rocm_rope* rope, const int32_t* positions,
                                 uint64_t rows, uint32_t head_dimension, const hllm_rocm_tensor* q,
                                 const hllm_rocm_tensor* q_out, const hllm_rocm_tensor* k,
                                 const hllm_rocm_tensor* k_out) {
  return guarded([&] {
    check_device(device);
    check_rows(rows);
    if (head_dimension < 16 || head_dimension > 256 || head_dimension % 16)
      refuse("the head dimension is a multiple of 16, at most 256");
    check_rope(rope, head_dimension);
    if (!k != !k_out) refuse("k and k_out come together");
    if (rows == 0) return;
    RotateArgs a{};
    a.q = tensor(q, "q", rows, head_dimension, false);
    a.q_out = tensor(q_out, "q_out", rows, head_dimension, true);
    if (q->dtype != q_out->dtype || q->heads != q_out->heads) refuse("q_out must have q's dtype and heads");
    check_in_place(q, q_out, rows);
    a.q_heads = (int32_t)q->heads;
    if (k) {
      a.k = tensor(k, "k", rows, head_dimension, false);
      a.k_out = tensor(k_out, "k_out", rows, head_dimension, true);
      if (k->dtype != q->dtype) refuse("q and k must have one dtype");
      if (k->dtype != k_out->dtype || k->heads != k_out->heads) refuse("k_out must have k's dtype and heads");
      check_in_place(k, k_out, rows);
      a.k_heads = (int32_t)k->heads;
    }
    a.lanes = (int32_t)head_dimension / 16;
    check_rotate_grid(rows, a);
    take_rope(rope, positions, a);
    if (k) {
      check_apart(q_out->data, "q_out", k_out->data, "k_out");
      check_apart(q_out->data, "q_out", k->data, "k");
      check_apart(k_out->data, "k_out", q->data, "q");
    }
    OnDevice on(device);
    launch_rotate(static_cast<hipStream_t>(stream), q->dtype, -1, (int)rows, a);
    HIP_CHECK(hipGetLastError());
  });
}

hllm_status hllm_rocm_kv_append(int32_t device, void* stream, const hllm_rocm_kv_pages* pages, const int32_t* slots,
                                uint64_t rows, const hllm_rocm_tensor* k, const hllm_rocm_tensor* v,
                                const hllm_rocm_rope* rope, const int32_t* positions, const hllm_rocm_tensor* q,
                                const hllm_rocm_tensor* q_out) {
  return guarded([&] {
    check_device(device);
    check_rows(rows);
    RotateArgs a{};
    a.pages = pages_of(pages);
    const uint64_t D = pages->head_dimension;
    if (rope) check_rope(rope, D);
    if (!q != !q_out) refuse("q and q_out come together");
    if (q && !rope) refuse("q is taken to be rotated: it needs rope");
    if (rows == 0) return;
    if (!slots) refuse("slots is null");
    a.slots = slots;
    a.k = tensor(k, "k", rows, D, false);
    a.v = tensor(v, "v", rows, D, false);
    if (k->heads != pages->kv_heads || v->heads != pages->kv_heads) refuse("k and v must have the cache's heads");
    if (k->dtype != v->dtype) refuse("k and v must have one dtype");
    a.k_heads = a.v_heads = (int32_t)pages->kv_heads;
    if (q) {
      a.q = tensor(q, "q", rows, D, false);
      a.q_out = tensor(q_out, "q_out", rows, D, true);
      if (q->dtype != k->dtype) refuse("q and k must have one dtype");
      if (q->dtype != q_out->dtype || q->heads != q_out->heads) refuse("q_out must have q's dtype and heads");
      check_in_place(q, q_out, rows);
      a.q_heads = (int32_t)q->heads;
    }
    a.lanes = (int32_t)D / 16;
    check_rotate_grid(rows, a);
    if (rope) take_rope(rope, positions, a);
    check_apart(pages->keys, "the cache's keys", pages->values, "values");
    check_apart(pages->keys, "the cache's keys", pages->key_scales, "key_scales");
    check_apart(pages->keys, "the cache's keys", pages->value_scales, "value_scales");
    check_apart(pages->values, "the cache's values", pages->key_scales, "key_scales");
    check_apart(pages->values, "the cache's values", pages->value_scales, "value_scales");
    check_apart(pages->key_scales, "the cache's key_scales", pages->value_scales, "value_scales");
    if (q) {
      check_apart(q_out->data, "q_out", k->data, "k");
      check_apart(q_out->data, "q_out", v->data, "v");
      check_apart(q_out->data, "q_out", pages->keys, "the cache's keys");
      check_apart(q_out->data, "q_out", pages->values, "the cache's values");
      check_apart(q_out->data, "q_out", pages->key_scales, "the cache's key_scales");
      check_apart(q_out->data, "q_out", pages->value_scales, "the cache's value_scales");
    }
    OnDevice on(device);
    launch_rotate(static_cast<hipStream_t>(stream), k->dtype, (int)pages->format, (int)rows, a);
    HIP_CHECK(hipGetLastError());
  });
}

hllm_status hllm_rocm_kv_read(int32_t device, void* stream, const hllm_rocm_kv_pages* pages, const int32_t* slots,
                              uint64_t rows, const hllm_rocm_tensor* k_out, const hllm_rocm_tensor* v_out) {
  return guarded([&] {
    check_device(device);
    check_rows(rows);
    ReadArgs a{};
    a.pages = pages_of(pages);
    if (rows == 0) return;
    if (!slots) refuse("slots is null");
    a.slots = slots;
    a.rows = (int32_t)rows;
    a.k = tensor(k_out, "k_out", rows, pages->head_dimension, true);
    a.v = tensor(v_out, "v_out", rows, pages->head_dimension, true);
    if (k_out->heads != pages->kv_heads || v_out->heads != pages->kv_heads) refuse("k_out and v_out must have the cache's heads");
    if (k_out->dtype != v_out->dtype) refuse("k_out and v_out must have one dtype");
    if (rows * pages->kv_heads * (pages->head_dimension / 4) > kMostBlocks * kThreads) refuse("too many rows for these heads");
    check_apart(k_out->data, "k_out", v_out->data, "v_out");
    OnDevice on(device);
    launch_kv_read(static_cast<hipStream_t>(stream), k_out->dtype, (int)pages->format, (int)pages->head_dimension, a);
    HIP_CHECK(hipGetLastError());
  });
}

}  // extern "C"

namespace {

// How a call's work is cut and what its workspace holds: each pair's cut, then outputs and statistics of
// two parts of each workgroup.
struct AttendPlan {
  uint64_t head_groups = 1, blocks = 0, cuts = 0, parts = 0, bytes = 0;
  bool shared = false;
};

AttendPlan plan_attention(const hllm_rocm_kv_pages& pages, uint64_t rows, uint64_t query_heads, uint64_t limit) {
  if (query_heads < 1 || query_heads > 1024 || query_heads % pages.kv_heads)
    refuse("query heads are a multiple of the cache's heads, at most 1024");
  AttendPlan p;
  if (rows == 0) return p;
  const uint64_t group = query_heads / pages.kv_heads;
  p.head_groups = (group + 15) / 16;
  const uint64_t pairs = rows * pages.kv_heads * p.head_groups, steps = (limit + 127) / 128, cost = kPairCost + steps;
  if (pairs > kMostBlocks) refuse("too many rows for these heads");
  // A workgroup for each pair where rows are short or pairs many: no row has more steps than 5 and 9 for each
  // pair a workgroup of the card. Shares cost 3 to 5 us more (each workgroup sums all rows' steps; the join), and
  // spare waiting for the longest row. Us with a pair each / with shares on either side of the line, BF16, 8 KV heads, groups of
  // 4, lengths log-uniform from 32:
  //   128: 16 rows to 768 11.8 / 11.8, to 1152 15.3 / 12.8; 64 rows to 1408 20.4 / 20.8, to 1920 24.7 / 22.8;
  //        256 rows to 1792 53.9 / 54.7, to 2688 71.9 / 70.3, to 3712 92.5 / 85.9, to 5120 117 / 102
  //   64:  16 rows to 768 9.4 / 10.1, to 1024 11.2 / 10.2; 64 rows to 1152 12.9 / 14.0, to 1664 16.7 / 15.8
  //   256: 16 rows to 896 18.0 / 16.1; 64 rows to 1280 29.4 / 31.8, to 1792 35.6 / 33.7, to 2432 44.2 / 37.6
  //   F32, 128: 64 rows to 1408 23.1 / 23.5, to 1920 28.4 / 26.0; F32, 256: 64 rows to 896 36.6 / 36.4, to 1792 53.0 / 46.4
  // So the crossing lies at the line for some tens of rows, and below it by a third for hundreds (the line loses up to 13%
  // there) and for F32 heads of 256. Rows that are padding count as pairs, for the host does not know them: 16
  // rows to 8000 take 21.8, with 48 padding rows 22.0, with 900, where pairs stay whole, 73.
  const uint64_t fit = attend_blocks((int)pages.head_dimension, false);
  const bool whole = steps * fit <= 5 * fit + 9 * pairs;
  p.blocks = pairs;
  if (whole || rows > kMostSharedRows) return p;
  // The line of all pairs is counted in 31 bits. Where it could be longer the pairs stay whole, but the
  // workspace is that of shares: a bound of the lengths is never given less than a smaller bound.
  p.shared = pairs <= (1u << 30) / cost;
  const uint64_t sharing = std::min<uint64_t>(fit, pairs * cost);
  if (p.shared) p.blocks = sharing;
  p.cuts = (pairs + 1) / 2 * 2;  // whole sixteen bytes
  p.parts = 2 * sharing * std::min<uint64_t>(group, 16);
  p.bytes = p.cuts * sizeof(int2) + p.parts * (pages.head_dimension + 2) * sizeof(float);
  return p;
}

// Positions of one row: sums of a length and a tile's stay below 2^31.
constexpr uint64_t kMostPositions = 1u << 30;

uint64_t clamp_length(uint64_t max_length) { return std::min(max_length, kMostPositions); }

}  // namespace

extern "C" {

hllm_status hllm_rocm_kv_attention_workspace(const hllm_rocm_kv_pages* pages, uint64_t rows, uint32_t query_heads,
                                             uint64_t max_length, uint64_t* bytes) {
  return guarded([&] {
    if (!bytes) refuse("null argument");
    pages_of(pages);
    check_rows(rows);
    *bytes = plan_attention(*pages, rows, query_heads, clamp_length(max_length)).bytes;
  });
}

hllm_status hllm_rocm_kv_attention(int32_t device, void* stream, const hllm_rocm_kv_pages* pages,
                                   const hllm_rocm_kv_attention_args* args) {
  return guarded([&] {
    check_device(device);
    AttendArgs a{};
    a.pages = pages_of(pages);
    if (!args) refuse("args is null");
    const uint64_t rows = args->rows, D = pages->head_dimension;
    check_rows(rows);
    if (rows == 0) return;
    a.q = tensor(&args->q, "q", rows, D, false);
    a.out = tensor(&args->out, "out", rows, D, true);
    if (args->q.dtype != args->out.dtype || args->q.heads != args->out.heads) refuse("out must have q's dtype and heads");
    if (args->q.data == args->out.data) refuse("out must not be q");
    if (!std::isfinite((float)(args->scale * kLog2e))) refuse("scale is not finite");  // as the kernels take it, with log2 e
    if (!args->lengths) refuse("lengths is null");
    if (args->table_width > kMostPositions / pages->page_tokens) refuse("a page table's row holds at most 2^30 positions");
    const uint64_t limit = std::min(clamp_length(args->max_length), args->table_width * pages->page_tokens);
    if (limit > 0 && !args->page_table) refuse("page_table is null");
    if (args->table_stride > (1ull << 40)) refuse("table_stride is too large");
    const AttendPlan plan = plan_attention(*pages, rows, args->q.heads, limit);
    if (plan.bytes > 0 && (!args->workspace || args->workspace_bytes < plan.bytes || (uintptr_t)args->workspace % 16))
      refuse("the workspace is null, not 16-byte aligned or below " + std::to_string(plan.bytes) + " bytes");
    if (plan.bytes > 0) {
      check_apart(args->workspace, "the workspace", args->out.data, "out");
      check_apart(args->workspace, "the workspace", args->q.data, "q");
    }
    a.table = args->page_table;
    a.table_stride = args->table_stride;
    a.lengths = args->lengths;
    a.rows = (int32_t)rows;
    a.q_heads = (int32_t)args->q.heads;
    a.group = a.q_heads / a.pages.kv_heads;
    a.head_groups = (int32_t)plan.head_groups;
    a.limit = (int32_t)limit;
    // F32 queries take twice the LDS.
    const bool f32 = args->q.dtype == HLLM_DTYPE_F32;
    a.blocks = (int32_t)(plan.shared ? std::min(plan.blocks, attend_blocks((int)D, f32)) : plan.blocks);
    a.shared = plan.shared;
    a.scale_hi = (float)(args->scale * kLog2e);
    a.scale_lo = (float)(args->scale * kLog2e - a.scale_hi);
    if (plan.shared) {
      a.cuts = static_cast<int2*>(args->workspace);
      a.part = reinterpret_cast<float*>(a.cuts + plan.cuts);
      a.stats = a.part + plan.parts * D;
    }
    OnDevice on(device);
    launch_kv_attention(static_cast<hipStream_t>(stream), args->q.dtype, (int)pages->format, (int)D, a);
    HIP_CHECK(hipGetLastError());
  });
}

}  // extern "C"
