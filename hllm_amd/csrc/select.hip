// The pages that a row's attention reads, selected by a cheap score: the bounds of pages' keys, the scores of a query against
// them and the selection. The C entry points are at the end.
#include <algorithm>

#include "operators_check.hpp"
#include "operators_device.hpp"

namespace hllm_rocm {
namespace {

typedef int32_t int4v __attribute__((ext_vector_type(4)));

// The biased exponent of the smallest power of two that leaves a magnitude (as bits, at least 2^-100) at most 127, which
// is 1.984375 * 2^6. Numbers times the power's inverse are exact, so what is rounded afterwards has one rounding.
__device__ inline uint32_t whole_power(uint32_t most) { return ((max(most, 27u << 23) + 0x1ffffu) >> 23) - 6; }

// Eight whole numbers as bytes.
__device__ inline uint2v bytes8(const int* x) {
  uint2v w;
#pragma unroll
  for (int j = 0; j < 2; ++j)
    w[j] = (x[4 * j] & 255) | (x[4 * j + 1] & 255) << 8 | (x[4 * j + 2] & 255) << 16 | (uint32_t)x[4 * j + 3] << 24;
  return w;
}

// ---------------------------------------------------------------- bounds

// Eight elements of a position's key as they are held.
template <int F, int D>
struct Keys8 {
  uint32_t codes[F < kE2m1 ? 2 : 1];
  uint32_t scale;
  __device__ void load(const Pages& c, const uint8_t* from, uint64_t vector, int d) {
    if constexpr (F < kE2m1) {
      const uint2v w = *reinterpret_cast<const uint2v*>(from + d);
      codes[0] = w[0], codes[1] = w[1];
      scale = static_cast<const uint32_t*>(c.key_scales)[vector];
    } else {
      codes[0] = *reinterpret_cast<const uint32_t*>(from + d / 2);
      const uint64_t group = vector * (D / 32) + d / 32;
      scale = F == kE2m1 ? static_cast<const uint8_t*>(c.key_scales)[group] : static_cast<const uint16_t*>(c.key_scales)[group];
    }
  }
  // What values() has to be multiplied by: exact where a bound's code is not 0, and infinite where the element is.
  static constexpr float kUnits = F == kInt4 ? 16.0f : 1.0f;
  // The elements in F32, over kUnits; false where they are not numbers (infinite ones show in their maximum).
  __device__ bool values(float* x) const {
    if constexpr (F == kE2m1) {
      const float by = __uint_as_float(scale << 23);
      const auto a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes[0], by, 0), b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes[0], by, 1),
                 c = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes[0], by, 2), d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes[0], by, 3);
      x[0] = a[0], x[1] = a[1], x[2] = b[0], x[3] = b[1], x[4] = c[0], x[5] = c[1], x[6] = d[0], x[7] = d[1];
      return scale != 255;
    } else if constexpr (F == kInt4) {
      // (n - 8) scale of four bits n, as one rounding of what F32 holds exactly, in sixteenths: 8 scale is past F32's range for scales
      // from 2^125 on, which keys of 2.98e38 are written with. (((float)n - 8) scale has an instruction more: 8 rows of 10000 positions,
      // 8 heads of 128, pages of 16, 20.6 us.)
      const float by = __uint_as_float(scale << 16) * (1.0f / kUnits);
      const uint32_t even = codes[0] & 0x0f0f0f0fu, odd = codes[0] >> 4 & 0x0f0f0f0fu;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        x[2 * i] = fmaf((float)(even >> (8 * i) & 255u), by, -8.0f * by);
        x[2 * i + 1] = fmaf((float)(odd >> (8 * i) & 255u), by, -8.0f * by);
      }
      return (scale & 0x7f80u) != 0x7f80u;
    } else {
      bool numbers = (scale & 0x7f800000u) != 0x7f800000u;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const floatx4 v = decode4<F>(codes[j]);
#pragma unroll
        for (int i = 0; i < 4; ++i) x[4 * j + i] = v[i] * __uint_as_float(scale);
        if constexpr (F == HLLM_KV_E4M3) numbers &= (((codes[j] & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u) == 0;
      }
      return numbers;
    }
  }
};

// Over the slots of a wave that hold other positions, eight channels each: the channels are parted among the slots in
// step with the maximum, so that a lane ends with 8 / slots channels (from `first` on) and half the work.
template <int L, typename Op>
__device__ inline void reduce_slots(float* x, Op&& op) {
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const auto both = __builtin_amdgcn_permlane32_swap(__float_as_uint(x[e]), __float_as_uint(x[e + 4]), false, false);
    x[e] = op(__uint_as_float(both[0]), __uint_as_float(both[1]));
  }
  if constexpr (L <= 16) {
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const auto both = __builtin_amdgcn_permlane16_swap(__float_as_uint(x[e]), __float_as_uint(x[e + 2]), false, false);
      x[e] = op(__uint_as_float(both[0]), __uint_as_float(both[1]));
    }
  }
  if constexpr (L == 8) {
    const bool upper = threadIdx.x & 8;
    const float send = upper ? x[0] : x[1];
    x[0] = op(upper ? x[1] : x[0],
              __uint_as_float((uint32_t)__builtin_amdgcn_update_dpp(0, (int)__float_as_uint(send), 0x128, 0xf, 0xf, false)));
  }
}

// The largest over the L lanes of a slot.
template <int L>
__device__ inline uint32_t slot_max(uint32_t v) {
  v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0xb1, 0xf, 0xf, false));   // the lane's pair's other
  v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x4e, 0xf, 0xf, false));   // of its four
  v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x141, 0xf, 0xf, false));  // of its eight
  if constexpr (L == 16) v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x140, 0xf, 0xf, false));  // of its sixteen
  return v;
}

// A page of a row, found from its place among the rows' `places`; false where there is nothing to make.
struct BoundsPage {
  int id, count;
  template <typename Load>
  __device__ bool find(const BoundsArgs& a, int row, int j, Load&& number) {
    const int shift = a.pages.page_shift, length = min(number(a.lengths + row), a.limit), start = max(number(a.starts + row), 0);
    const int p = (start >> shift) + j;
    if (start >= length || p > (length - 1) >> shift) return false;
    id = number(a.table + (uint64_t)row * a.table_stride + p);
    count = min(1 << shift, length - (p << shift));
    return id >= 0 && id < a.pages.pages;
  }
};

// A page and KV head for each slot of L lanes, a lane eight channels of all positions: nothing is exchanged between lanes but the
// largest magnitude. For many short pages. Bound by its reads where it is at its best: 8 rows of 10000 positions, 8 KV heads of 128, E2M1,
// pages of 16: 14.5 us, 3.7 TB/s of what is read and written.
template <int F, int D>
__global__ void __launch_bounds__(kThreads) kv_bounds_slots_kernel(BoundsArgs a) {
  constexpr int L = D / 8, S = 64 / L, kDeep = 8;
  const Pages& c = a.pages;
  const uint32_t item = (blockIdx.x * 4 + (threadIdx.x >> 6)) * S + (threadIdx.x & 63) / L;
  const uint32_t place = item / (uint32_t)c.kv_heads, row = place / (uint32_t)a.places;
  const int h = (int)(item - place * c.kv_heads), d = (int)(threadIdx.x % L) * 8;
  BoundsPage page;
  if (row >= (uint32_t)a.rows || !page.find(a, (int)row, (int)(place - row * a.places), [](const int32_t* at) { return *at; })) return;
  const uint8_t* from = c.keys + (uint64_t)page.id * c.page_stride + (uint64_t)h * c.head_stride;
  const uint64_t own = (uint64_t)page.id * c.kv_heads + h, vector = own << c.page_shift;
  Keys8<F, D> k[kDeep];
  const auto load = [&](int t) {
#pragma unroll
    for (int i = 0; i < kDeep; ++i) {
      const int at = min(t + i, page.count - 1);  // the last position again changes nothing
      k[i].load(c, from + (uint64_t)(uint32_t)at * c.token_stride, vector + at, d);
    }
  };
  float high[8], low[8];
  bool numbers = true;
#pragma unroll
  for (int i = 0; i < 8; ++i) high[i] = -INFINITY, low[i] = INFINITY;
  load(0);
  for (int t = 0; t < page.count; t += kDeep) {
    Keys8<F, D> now[kDeep];
#pragma unroll
    for (int i = 0; i < kDeep; ++i) now[i] = k[i];
    if (t + kDeep < page.count) load(t + kDeep);
#pragma unroll
    for (int i = 0; i < kDeep; i += 2) {
      float x[8], y[8];
      numbers &= now[i].values(x);
      numbers &= now[i + 1].values(y);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        high[e] = fmaxf(fmaxf(high[e], x[e]), y[e]);
        low[e] = fminf(fminf(low[e], x[e]), y[e]);
      }
    }
  }
  uint32_t most = numbers ? 0u : 0x7f800000u;
#pragma unroll
  for (int e = 0; e < 8; ++e) high[e] *= Keys8<F, D>::kUnits, low[e] *= Keys8<F, D>::kUnits;
#pragma unroll
  for (int e = 0; e < 8; ++e) most = max(most, max(__float_as_uint(high[e]) & 0x7fffffffu, __float_as_uint(low[e]) & 0x7fffffffu));
  most = slot_max<L>(most);
  const bool bad = most >= 0x7f800000u;
  const uint32_t power = whole_power(most);
  const float inverse = __uint_as_float((254u - power) << 23);
  int x[2][8];
#pragma unroll
  for (int e = 0; e < 8; ++e) x[0][e] = bad ? 0 : (int)rintf(high[e] * inverse), x[1][e] = bad ? 0 : (int)rintf(low[e] * inverse);
#pragma unroll
  for (int which = 0; which < 2; ++which) *reinterpret_cast<uint2v*>(a.codes + (own * 2 + which) * D + d) = bytes8(x[which]);
  if (d == 0) a.scales[own] = bad ? NAN : __uint_as_float(power << 23);
}

// A wave (kWaves = 1) or a workgroup's four for a page and KV head, for few pages or long ones: a lane has
// eight channels of every (D = 64: eighth, 128: fourth, 256: second) position. The next positions are under way while some are
// compared. After one token a row it is a launch and a chain of row, page, keys: 32 rows of 8 heads of 128 in pages of 16 2.6 us. Prompts in
// long pages are bound by their reads: 8 rows of 10000 positions, 4 heads of 256, INT8, pages of 64: 22.1 us, 3.9 TB/s.
template <int F, int D, int kWaves>
__global__ void __launch_bounds__(kThreads) kv_bounds_kernel(BoundsArgs a) {
  constexpr int L = D / 8, S = 64 / L, C = 8 / S, kDeep = 4;  // lanes of a vector, positions at once, channels left, loads in flight
  __shared__ float meet[kWaves > 1 ? kWaves : 1][2][kWaves > 1 ? D : 1];
  __shared__ int spoiled[kWaves];
  const Pages& c = a.pages;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const uint32_t item = kWaves > 1 ? blockIdx.x : blockIdx.x * 4 + wave;
  const uint32_t place = item / (uint32_t)c.kv_heads, row = place / (uint32_t)a.places;
  const int h = (int)(item - place * c.kv_heads), slot = lane / L, d = lane % L * 8;
  BoundsPage page;
  if (row >= (uint32_t)a.rows || !page.find(a, (int)row, (int)(place - row * a.places), [](const int32_t* at) { return uniform_load(at); })) return;
  const uint8_t* from = c.keys + (uint64_t)page.id * c.page_stride + (uint64_t)h * c.head_stride;
  const uint64_t own = (uint64_t)page.id * c.kv_heads + h, vector = own << c.page_shift;
  Keys8<F, D> k[kDeep];
  const auto load = [&](int t) {
#pragma unroll
    for (int i = 0; i < kDeep; ++i) {
      const int at = min(t + i * S + slot, page.count - 1);  // the last position again changes nothing
      k[i].load(c, from + (uint64_t)(uint32_t)at * c.token_stride, vector + at, d);
    }
  };
  float high[8], low[8];
  bool numbers = true;
#pragma unroll
  for (int i = 0; i < 8; ++i) high[i] = -INFINITY, low[i] = INFINITY;
  constexpr int kStep = kWaves * S * kDeep;
  const int first = kWaves > 1 ? wave * S * kDeep : 0;
  load(first);
  for (int t = first; t < page.count; t += kStep) {
    Keys8<F, D> now[kDeep];
#pragma unroll
    for (int i = 0; i < kDeep; ++i) now[i] = k[i];
    if (t + kStep < page.count) load(t + kStep);
#pragma unroll
    for (int i = 0; i < kDeep; i += 2) {
      float x[8], y[8];
      numbers &= now[i].values(x);
      numbers &= now[i + 1].values(y);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        high[e] = fmaxf(fmaxf(high[e], x[e]), y[e]);
        low[e] = fminf(fminf(low[e], x[e]), y[e]);
      }
    }
  }
  reduce_slots<L>(high, [](float x, float y) { return fmaxf(x, y); });
  reduce_slots<L>(low, [](float x, float y) { return fminf(x, y); });
  bool bad = __any(!numbers);
  const int channel = d + (lane & 32 ? 4 : 0) + (L <= 16 && (lane & 16) ? 2 : 0) + (L == 8 && (lane & 8) ? 1 : 0);
  if constexpr (kWaves > 1) {
#pragma unroll
    for (int e = 0; e < C; ++e) meet[wave][0][channel + e] = high[e], meet[wave][1][channel + e] = low[e];
    if (lane == 0) spoiled[wave] = bad;
    __syncthreads();
    if (wave > 0) return;
#pragma unroll
    for (int w = 1; w < kWaves; ++w) {
      bad |= spoiled[w] != 0;
#pragma unroll
      for (int e = 0; e < C; ++e) high[e] = fmaxf(high[e], meet[w][0][channel + e]), low[e] = fminf(low[e], meet[w][1][channel + e]);
    }
  }
  uint32_t most = 0;
#pragma unroll
  for (int e = 0; e < C; ++e) high[e] *= Keys8<F, D>::kUnits, low[e] *= Keys8<F, D>::kUnits;
#pragma unroll
  for (int e = 0; e < C; ++e) most = max(most, max(__float_as_uint(high[e]) & 0x7fffffffu, __float_as_uint(low[e]) & 0x7fffffffu));
  most = wave_max(most);
  bad |= most >= 0x7f800000u;
  const uint32_t power = whole_power(most);
  const float inverse = __uint_as_float((254u - power) << 23);
  uint32_t codes[2] = {0, 0};
#pragma unroll
  for (int e = 0; e < C; ++e) {
    codes[0] |= ((uint32_t)(int)rintf(high[e] * inverse) & 255u) << (8 * e);
    codes[1] |= ((uint32_t)(int)rintf(low[e] * inverse) & 255u) << (8 * e);
  }
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    int8_t* to = a.codes + (own * 2 + which) * D + channel;
    const uint32_t w = bad ? 0u : codes[which];
    if constexpr (C == 1) *reinterpret_cast<uint8_t*>(to) = (uint8_t)w;
    if constexpr (C == 2) *reinterpret_cast<uint16_t*>(to) = (uint16_t)w;
    if constexpr (C == 4) *reinterpret_cast<uint32_t*>(to) = w;
  }
  if (lane == 0) a.scales[own] = bad ? NAN : __uint_as_float(power << 23);
}

// ---------------------------------------------------------------- scores

// Numbers' bits so that whole numbers order as the numbers do, -0 as 0; NaN is above all of them.
constexpr uint32_t kNoNumber = 0xfffffffeu;
__device__ inline uint32_t ordered(float x) {
  const uint32_t bits = __float_as_uint(x + 0.0f);
  return bits ^ ((uint32_t)((int)bits >> 31) | 0x80000000u);
}

// The largest over the sixteen lanes of a row.
template <int O>
__device__ inline float row_max(float v) {
  return fmaxf(v, __uint_as_float((uint32_t)__builtin_amdgcn_update_dpp(0, (int)__float_as_uint(v), 0x120 + O, 0xf, 0xf, false)));
}

// Sixteen queries as whole numbers, positive and negative elements apart, and their powers of two.
template <int D>
struct Queries {
  uint2v up[16][D / 8], down[16][D / 8];
  float scale[16];
};

// The scores of a row's pages for one KV head, as ordered whole numbers: keep(page's place, number, whether it is another
// sixteen query heads' and the larger counts). Every thread of a workgroup of kWaves waves is here. A wave takes kPages pages at once, from
// kPages `first` on in steps of `step`. With a query's positive and negative elements apart, the sum over channels of the
// larger product is one product [high, low] x [max(q, 0), min(q, 0)] of twice the length, on the matrix units in
// bytes, with the query heads of a KV head as columns. Sums of whole numbers below 2^24 and powers of two are exact. The first
// bounds are under way while the workgroup rounds the queries, and the next ones while some are multiplied (32 rows of 1200 pages of 8 heads of
// 128: 23.8 us, 26.0 without; 128 of 1000: 87, 95).
template <int D>
constexpr int kScorePages = D == 64 ? 64 : D == 128 ? 32 : 16;
template <typename T, int D, int kWaves, typename Keep>
__device__ inline void score_pages(const SelectArgs& a, Queries<D>& queries, int row, int kvh, int count, int first, int step,
                                   Keep&& keep) {
  constexpr int KK = D / 64, kPages = kScorePages<D>, kTiles = kPages / 16;
  const int lane = threadIdx.x & 63, quad = lane >> 4, col = lane & 15;
  const int32_t* table = a.table + (uint64_t)row * a.table_stride;
  int4v high[kTiles][KK], low[kTiles][KK];
  float scale = 0.0f;    // of the lane's page
  bool absent = false;   // whether it is outside the cache
  int id = 0;            // the page of the next load
  const auto find = [&](int t) { id = table[min(t + lane % kPages, count - 1)]; };
  const auto load = [&](int t) {
    absent = id < 0 || id >= a.pages;
    const int own = absent ? 0 : id;
    scale = a.scales[(uint64_t)own * a.kv_heads + kvh];
#pragma unroll
    for (int i = 0; i < kTiles; ++i) {
      const uint64_t page = (uint64_t)__shfl(own, 16 * i + col, 64) * a.kv_heads + kvh;
      const int8_t* from = a.codes + page * (2 * D) + 16 * quad;
#pragma unroll
      for (int kk = 0; kk < KK; ++kk) {
        high[i][kk] = *reinterpret_cast<const int4v*>(from + 64 * kk);
        low[i][kk] = *reinterpret_cast<const int4v*>(from + D + 64 * kk);
      }
    }
    if (t + kPages * step < count) find(t + kPages * step);
  };
  for (int g0 = 0; g0 < a.group; g0 += 16) {
    const int vectors = min(16, a.group - g0);
    int t = kPages * first;
    if (t < count) find(t), load(t);
    if (g0 > 0) __syncthreads();
    // D / 8 threads a query; queries behind the last repeat it.
    constexpr int kEach = D / 8;
#pragma unroll
    for (int at = 0; at < 16 * kEach; at += 64 * kWaves) {
      const int of = (at + (int)threadIdx.x) / kEach, u = (at + (int)threadIdx.x) % kEach;
      if (16 * kEach < 64 * kWaves && of >= 16) break;  // whole waves
      float x[8];
      load8(hllm_rocm::at<const T>(a.q, row, kvh * a.group + g0 + min(of, vectors - 1), 8 * u), x);
      uint32_t most = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) most = max(most, __float_as_uint(x[i]) & 0x7fffffffu);
#pragma unroll
      for (int o = 1; o < kEach; o <<= 1) most = max(most, (uint32_t)__shfl_xor((int)most, o, 64));
      const bool finite = most < 0x7f800000u;
      const uint32_t power = whole_power(most);
      const float inverse = __uint_as_float((254u - power) << 23);
      int p[8], n[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int v = finite ? (int)rintf(x[i] * inverse) : 0;
        p[i] = max(v, 0);
        n[i] = min(v, 0);
      }
      queries.up[of][u] = bytes8(p);
      queries.down[of][u] = bytes8(n);
      if (u == 0) queries.scale[of] = finite ? __uint_as_float(power << 23) : NAN;
    }
    __syncthreads();
    int4v up[KK], down[KK];
#pragma unroll
    for (int kk = 0; kk < KK; ++kk) {
      up[kk] = *reinterpret_cast<const int4v*>(&queries.up[col][8 * kk + 2 * quad]);
      down[kk] = *reinterpret_cast<const int4v*>(&queries.down[col][8 * kk + 2 * quad]);
    }
    const float q_scale = queries.scale[col];
    const bool no_query = __any(q_scale != q_scale);
    for (; t < count; t += kPages * step) {
      int4v high_now[kTiles][KK], low_now[kTiles][KK];
#pragma unroll
      for (int i = 0; i < kTiles; ++i)
#pragma unroll
        for (int kk = 0; kk < KK; ++kk) high_now[i][kk] = high[i][kk], low_now[i][kk] = low[i][kk];
      const float scale_now = scale;
      const bool absent_now = absent;
      if (t + kPages * step < count) load(t + kPages * step);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int i = 0; i < kTiles; ++i) {
        int4v dot = {0, 0, 0, 0};
#pragma unroll
        for (int kk = 0; kk < KK; ++kk) {
          dot = __builtin_amdgcn_mfma_i32_16x16x64_i8(high_now[i][kk], up[kk], dot, 0, 0, 0);
          dot = __builtin_amdgcn_mfma_i32_16x16x64_i8(low_now[i][kk], down[kk], dot, 0, 0, 0);
        }
        float mine = 0.0f;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float v = row_max<1>(row_max<2>(row_max<4>(row_max<8>((float)dot[e] * q_scale))));
          mine = col == e ? v : mine;
        }
        // A lane of the first four of its row has the page 16 i + 4 quad + col; a page's scale does not change which head is the largest.
        const int of = 16 * i + 4 * quad + (col & 3), place = t + of;
        const float by = __shfl(scale_now, of, 64);
        const bool gone = __shfl((int)absent_now, of, 64);
        uint32_t key = by != by || no_query ? kNoNumber : ordered(mine * by);
        if (gone) key = 0;
        if (col < 4 && place < count) keep(place, key, g0 > 0);
      }
    }
  }
}

__device__ inline int pages_of(const SelectArgs& a, int row, int& length) {
  length = min(uniform_load(a.lengths + row), a.limit);
  return length <= 0 ? 0 : ((length - 1) >> a.page_shift) + 1;
}

// Scores into the workspace, for rows of more pages than one workgroup scores. 32 rows of 4000 pages, 8 heads of 128 (266 MB of bounds):
// 83 us with the selection, the bounds read at 3.8 TB/s, 5.3 with the lines of the pages' scales, of which a KV head uses four bytes. A row's heads
// on one die, which then reads those lines once, take 81 to 83; pages in order 80.
template <typename T, int D>
__global__ void __launch_bounds__(kThreads, 4) kv_score_kernel(SelectArgs a) {
  const int row = blockIdx.x / a.kv_heads, kvh = blockIdx.x % a.kv_heads;
  int length;
  const int count = pages_of(a, row, length);
  if (count <= a.keep) return;
  __shared__ Queries<D> queries;
  uint32_t* keys = a.keys + (uint64_t)blockIdx.x * a.stride;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  // Workgroups without a page: every other takes the queries' barriers.
  if ((int)blockIdx.y * 4 * kScorePages<D> >= count) return;
  score_pages<T, D, 4>(a, queries, row, kvh, count, blockIdx.y * 4 + wave, gridDim.y * 4,
                    [&](int place, uint32_t key, bool again) { keys[place] = again ? max(keys[place], key) : key; });
}

// ---------------------------------------------------------------- selection

// How a selection is made: by workgroups of four or of sixteen waves that score their pages themselves, or by ones of sixteen
// waves whose pages others have scored. Threads, and scores that each holds at once.
enum Select { kSmall, kLarge, kScored };
template <Select kHow>
constexpr int kSelectThreads = kHow == kSmall ? 256 : 1024;
template <Select kHow>
constexpr int kSelectOwn = kHow == kSmall ? 2 : kHow == kLarge ? 4 : 16;
constexpr int kDigit = 11;  // bits that a pass over the scores settles

// A workgroup selects a row's pages for one KV head. Passes over the scores, upper bits first, count how many there are of each value of
// the next bits among those that may still be the last one selected; then the pages above it are written, and of those at
// it the first ones, in their order. A selection by itself takes some 8 us, five barriers of sixteen waves a pass over eleven bits; with its
// scores 32 rows of 12000 to 30000 positions in pages of 16, 8 heads of 128, 33 us: the longest row's workgroup, alone on its CU.
template <typename T, int D, Select kHow>
__global__ void __launch_bounds__(kSelectThreads<kHow>) kv_select_kernel(SelectArgs a) {
  constexpr bool kHere = kHow != kScored;
  constexpr int kThreadsHere = kSelectThreads<kHow>, W = kThreadsHere / 64, kOwn = kSelectOwn<kHow>;
  constexpr int kTile = kThreadsHere * kOwn, kBins = 1 << kDigit, kEach = kBins / kThreadsHere;
  __shared__ uint32_t scored[kHere ? kTile : 1];
  __shared__ int bins[kBins];
  __shared__ uint32_t range[W][2];
  __shared__ int sums[W], found[3];
  __shared__ int before[kOwn * W];
  const int row = blockIdx.x / a.kv_heads, kvh = blockIdx.x % a.kv_heads;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  int length;
  const int n = pages_of(a, row, length);
  if (kvh == 0 && threadIdx.x == 0)
    a.selected_lengths[row] = n <= a.keep ? length : length - ((n - a.keep) << a.page_shift);
  if (length < 0) return;  // a padding row's pages are left
  const int32_t* table = a.table + (uint64_t)row * a.table_stride;
  int32_t* out = a.selected + (uint64_t)blockIdx.x * a.keep;
  if (n <= a.keep) {
    for (int i = threadIdx.x; i < a.keep; i += kThreadsHere) out[i] = i < n ? table[i] : -1;
    return;
  }
  const uint32_t* keys = a.keys + (uint64_t)blockIdx.x * a.stride;
  if constexpr (kHere) {
    __shared__ Queries<D> queries;
    score_pages<T, D, W>(a, queries, row, kvh, n, wave, W,
                         [&](int place, uint32_t key, bool again) { scored[place] = again ? max(scored[place], key) : key; });
    __syncthreads();
  }
  // A thread's scores of a tile: of places from + j * kThreadsHere. `open` has a bit for each that is selected by its score.
  const int tiles = (n + kTile - 1) / kTile;
  uint32_t v[kOwn], open = 0;
  int ids[kOwn], used = 0;
  const auto load = [&](int tile) {
    const int from = tile * kTile + (int)threadIdx.x;
    used = min(kOwn, (n - tile * kTile + kThreadsHere - 1) / kThreadsHere);
    open = 0;
#pragma unroll
    for (int j = 0; j < kOwn; ++j) {
      const int i = from + j * kThreadsHere;
      v[j] = 0;
      if (j < used && i < n) {
        if (i >= a.first && i < n - a.last) open |= 1u << j;
        v[j] = kHere ? scored[i] : keys[i];
        ids[j] = table[i];
      }
    }
  };
  uint32_t all = 0xffffffffu, some = 0;
  for (int tile = 0; tile < tiles; ++tile) {
    load(tile);
#pragma unroll
    for (int j = 0; j < kOwn; ++j)
      if (open >> j & 1) all &= v[j], some |= v[j];
  }
  for (int o = 1; o < 64; o <<= 1) {
    all &= (uint32_t)__shfl_xor((int)all, o, 64);
    some |= (uint32_t)__shfl_xor((int)some, o, 64);
  }
  if (lane == 0) range[wave][0] = all, range[wave][1] = some;
  __syncthreads();
  all = range[lane % W][0], some = range[lane % W][1];
  for (int o = 1; o < W; o <<= 1) {
    all &= (uint32_t)__shfl_xor((int)all, o, 64);
    some |= (uint32_t)__shfl_xor((int)some, o, 64);
  }
  // The scores that are open are those whose upper bits, from `bits` on, are `prefix`; `need` of them are to be selected.
  int bits = all == some ? 0 : 32 - __builtin_clz(all ^ some), need = a.keep - a.first - a.last;
  uint64_t prefix = (uint64_t)all >> bits;
  bool whole = need == 0;  // all that are left are selected, or (none needed) none
  if (whole) prefix = ~0ull;
  while (bits > 0 && !whole) {
    const int shift = max(bits - kDigit, 0), mask = (1 << (bits - shift)) - 1;
#pragma unroll
    for (int i = 0; i < kEach; ++i) bins[i * kThreadsHere + threadIdx.x] = 0;
    __syncthreads();
    for (int tile = 0; tile < tiles; ++tile) {
      if (tiles > 1) load(tile);
#pragma unroll
      for (int j = 0; j < kOwn; ++j)
        if ((open >> j & 1) && (uint64_t)v[j] >> bits == prefix) atomicAdd(&bins[v[j] >> shift & mask], 1);
    }
    __syncthreads();
    // Bins from the largest down: a thread's kEach, and how many scores the threads before it have.
    const int top = kBins - 1 - (int)threadIdx.x * kEach;
    int own = 0, sum;
#pragma unroll
    for (int i = 0; i < kEach; ++i) own += bins[top - i];
    sum = wave_scan(own, lane, 64);
    if (lane == 63) sums[wave] = sum;
    __syncthreads();
    int earlier = lane < wave ? sums[lane] : 0;
    for (int o = 1; o < W; o <<= 1) earlier += __shfl_xor(earlier, o, 64);
    sum += __builtin_amdgcn_readfirstlane(earlier);
    if (sum >= need && sum - own < need) {
      int above = sum - own, i = 0;
      while (above + bins[top - i] < need) above += bins[top - i++];
      found[0] = top - i, found[1] = need - above, found[2] = bins[top - i];
    }
    __syncthreads();
    prefix = prefix << (bits - shift) | (uint32_t)found[0];
    need = found[1];
    whole = need == found[2];
    bits = shift;
  }
  const int take = whole ? 0x7fffffff : need;  // of those at the prefix
  int larger = 0, equal = 0;  // of the tiles before
  for (int tile = 0; tile < tiles; ++tile) {
    if (tiles > 1) load(tile);
    uint32_t gt = 0, eq = 0;
    __syncthreads();
#pragma unroll
    for (int j = 0; j < kOwn; ++j) {
      if (j < used) {
        const int i = tile * kTile + j * kThreadsHere + (int)threadIdx.x;
        const uint64_t upper = (uint64_t)v[j] >> bits;
        const bool is_open = open >> j & 1, g = i < n && (!is_open || upper > prefix), e = is_open && upper == prefix;
        gt |= (uint32_t)g << j;
        eq |= (uint32_t)e << j;
        const int counts = __popcll(__ballot(g)) | __popcll(__ballot(e)) << 16;
        if (lane == 0) before[j * W + wave] = counts;
      }
    }
    __syncthreads();
    // How many lie before each wave's places: an exclusive sum over the places in their order.
    int total = 0;
    if (wave == 0) {
      for (int at = 0; at < used * W; at += 64) {
        const int own = at + lane < used * W ? before[at + lane] : 0;
        const int sum = wave_scan(own, lane, 64) + total;
        if (at + lane < used * W) before[at + lane] = sum - own;
        total = __builtin_amdgcn_readlane(sum, 63);
      }
      if (lane == 0) found[0] = total;
    }
    __syncthreads();
    const uint64_t lower = (1ull << lane) - 1;
#pragma unroll
    for (int j = 0; j < kOwn; ++j) {
      if (j < used) {
        const int at = before[j * W + wave];
        const int g = larger + (at & 0xffff) + __popcll(__ballot(gt >> j & 1) & lower);
        const int e = equal + (at >> 16) + __popcll(__ballot(eq >> j & 1) & lower);
        if ((gt >> j & 1) || ((eq >> j & 1) && e < take)) out[g + min(e, take)] = ids[j];
      }
    }
    larger += found[0] & 0xffff;
    equal += found[0] >> 16;
  }
}

template <int F>
void bounds_format(hipStream_t stream, int head_dim, const BoundsArgs& a) {
  const unsigned items = (unsigned)a.rows * a.places * a.pages.kv_heads;
  const auto run = [&](auto dim) {
    constexpr int D = decltype(dim)::value;
    constexpr unsigned kSlots = 4 * 512 / D;  // of a workgroup
    if (a.by == kByWorkgroup) kv_bounds_kernel<F, D, 4><<<items, kThreads, 0, stream>>>(a);
    if (a.by == kByWave) kv_bounds_kernel<F, D, 1><<<(items + 3) / 4, kThreads, 0, stream>>>(a);
    if constexpr (D <= 128)
      if (a.by == kBySlot) kv_bounds_slots_kernel<F, D><<<(items + kSlots - 1) / kSlots, kThreads, 0, stream>>>(a);
  };
  if (head_dim == 64) run(std::integral_constant<int, 64>{});
  if (head_dim == 128) run(std::integral_constant<int, 128>{});
  if (head_dim == 256) run(std::integral_constant<int, 256>{});
}

void launch_bounds(hipStream_t stream, int format, int head_dim, const BoundsArgs& a) {
  if (format == HLLM_KV_E4M3) return bounds_format<HLLM_KV_E4M3>(stream, head_dim, a);
  if (format == HLLM_KV_INT8) return bounds_format<HLLM_KV_INT8>(stream, head_dim, a);
  if (format == kE2m1) return bounds_format<kE2m1>(stream, head_dim, a);
  bounds_format<kInt4>(stream, head_dim, a);
}

template <typename T, int D>
void select_dim(hipStream_t stream, Select how, int chunks, const SelectArgs& a) {
  const unsigned pairs = (unsigned)(a.rows * a.kv_heads);
  if (how == kSmall) kv_select_kernel<T, D, kSmall><<<pairs, kSelectThreads<kSmall>, 0, stream>>>(a);
  if (how == kLarge) kv_select_kernel<T, D, kLarge><<<pairs, kSelectThreads<kLarge>, 0, stream>>>(a);
  if (how == kScored) {
    kv_score_kernel<T, D><<<dim3(pairs, chunks), kThreads, 0, stream>>>(a);
    kv_select_kernel<T, D, kScored><<<pairs, kSelectThreads<kScored>, 0, stream>>>(a);
  }
}

void launch_select(hipStream_t stream, uint32_t dtype, int head_dim, Select how, int chunks, const SelectArgs& a) {
  const auto run = [&](auto zero) {
    using T = decltype(zero);
    if (head_dim == 64) select_dim<T, 64>(stream, how, chunks, a);
    if (head_dim == 128) select_dim<T, 128>(stream, how, chunks, a);
    if (head_dim == 256) select_dim<T, 256>(stream, how, chunks, a);
  };
  if (dtype == HLLM_DTYPE_F16) return run(_Float16{});
  if (dtype == HLLM_DTYPE_BF16) return run(bhalf{});
  run(0.0f);
}

// ---------------------------------------------------------------- argument checks

int shift_of(uint32_t page_tokens) { return __builtin_ctz(page_tokens); }

void check_bounds(const hllm_rocm_kv_bounds* b) {
  if (!b) refuse("bounds is null");
  if (b->head_dimension != 64 && b->head_dimension != 128 && b->head_dimension != 256)
    refuse("a cache's head dimension is 64, 128 or 256");
  if (b->kv_heads < 1 || b->kv_heads > 1024) refuse("1 to 1024 key-value heads");
  if (b->page_tokens < 8 || b->page_tokens > 4096 || (b->page_tokens & (b->page_tokens - 1)))
    refuse("a page's tokens are a power of two, 8 to 4096");
  if (b->pages < 1 || (uint64_t)b->pages * b->page_tokens > 0x7fffffffull) refuse("a cache has 1 to 2^31 - 1 slots");
  if (!b->codes || !b->scales) refuse("the bounds' memory is null");
  if (((uintptr_t)b->codes | (uintptr_t)b->scales) % 16) refuse("the bounds' memory must be 16-byte aligned");
  check_apart(b->codes, "the bounds' codes", b->scales, "scales");
}

uint64_t table_positions(uint64_t width, uint64_t stride, uint32_t page_tokens) {
  if (width > kMostPositions / page_tokens) refuse("a page table's row holds at most 2^30 positions");
  if (stride > (1ull << 40)) refuse("table_stride is too large");
  return width * page_tokens;
}

void update_bounds(int32_t device, void* stream, const Cache& cache, const hllm_rocm_kv_bounds* bounds,
                   const hllm_rocm_kv_bounds_args* args) {
  check_bounds(bounds);
  if (!args) refuse("args is null");
  const Pages& pages = cache.pages;
  if ((int32_t)bounds->pages != pages.pages || bounds->page_tokens != cache.page_tokens ||
      (int32_t)bounds->kv_heads != pages.kv_heads || (int32_t)bounds->head_dimension != cache.head_dim)
    refuse("the bounds are those of another cache");
  check_rows(args->rows);
  const uint64_t positions = table_positions(args->table_width, args->table_stride, cache.page_tokens);
  const uint64_t fresh = std::min(args->max_new, positions);
  if (args->rows == 0 || fresh == 0) return;
  if (!args->page_table) refuse("page_table is null");
  if (!args->starts || !args->lengths) refuse("starts or lengths is null");
  for (const void* from : {(const void*)pages.keys, (const void*)pages.key_scales}) {
    check_apart(bounds->codes, "the bounds' codes", from, "the cache");
    check_apart(bounds->scales, "the bounds' scales", from, "the cache");
  }
  BoundsArgs a{};
  a.pages = pages;
  a.codes = bounds->codes;
  a.scales = bounds->scales;
  a.table = args->page_table;
  a.table_stride = args->table_stride;
  a.starts = args->starts;
  a.lengths = args->lengths;
  a.rows = (int32_t)args->rows;
  a.limit = (int32_t)positions;
  // `fresh` positions lie in this many pages at most.
  const uint64_t places = std::min<uint64_t>((fresh + 2 * cache.page_tokens - 2) / cache.page_tokens, args->table_width);
  a.places = (int32_t)places;
  const uint64_t items = args->rows * places * pages.kv_heads;
  if (args->rows * places > kMostBlocks || items > kMostBlocks) refuse("too many rows for these pages and heads");
  // Long pages, and pages that a lone wave reads in many steps where there are few of them (9 rows of 4 heads of 256 in pages of 64:
  // 5.5 us with a wave a page and head).
  const uint64_t loads = (uint64_t)cache.page_tokens * (cache.head_dim / 8) / 64;  // of a wave for a page and head
  // Many short pages: a slot of a wave each, for the maxima over a wave's slots take as long as a short page's elements. Us by waves / by slots:
  //   E2M1, 128, pages of 16: 1024 items 3.0 / 3.8, 4096 4.1 / 4.0, 8192 6.5 / 5.5, 40000 20.7 / 14.5; of 32: 20032 14.9 / 12.4; E4M3,
  //   64, of 16: 4096 4.2 / 4.6, 40000 21.9 / 11.5; E2M1, 64, of 8: 32768 16.9 / 6.1; INT8, 128, of 16: 40000 25.1 / 23.2, of 32: 20032
  //   21.6 / 21.8; longer pages and 256: INT4, 128, of 64: 10048 17.1 / 18.6; E2M1, 64, of 64: 10048 9.2 / 9.9; E4M3, 256, of 16: 20000 22.8 / 23.4
  a.by = cache.page_tokens > 128 || (items <= 1024 && loads > 4)                        ? kByWorkgroup
         : cache.page_tokens <= 32 && cache.head_dim <= 128 && items >= 8192            ? kBySlot
                                                                                        : kByWave;
  OnDevice on(device);
  launch_bounds(static_cast<hipStream_t>(stream), cache.format, cache.head_dim, a);
  HIP_CHECK(hipGetLastError());
}

// How a call's rows are scored and selected, and by how many workgroups a row and KV head they are scored (kScored).
struct SelectPlan {
  uint64_t limit = 0, stride = 0, bytes = 0;
  Select how = kSmall;
  int chunks = 0;
};

uint64_t score_pages_of(uint32_t head_dim) { return head_dim == 256 ? kScorePages<256> : head_dim == 128 ? kScorePages<128> : kScorePages<64>; }

SelectPlan plan_select(const hllm_rocm_kv_bounds& b, uint64_t rows, uint64_t max_length, uint64_t keep) {
  SelectPlan p;
  p.limit = std::min(max_length, kMostPositions);
  const uint64_t pages = (p.limit + b.page_tokens - 1) / b.page_tokens, pairs = rows * b.kv_heads;
  if (pairs > kMostBlocks) refuse("too many rows for these heads");
  if (rows == 0 || pages <= keep) return p;
  if (pages <= (uint64_t)kSelectThreads<kSmall> * kSelectOwn<kSmall>) return p;
  // With few pages, or workgroups for half the card, one launch takes less time than two. Us with workgroups that score
  // their own pages / with others that do, 8 KV heads of 128 and all rows of as many pages of 16:
  //   1 row: 600 pages 15.6 / 16.2, 1000 19.9 / 16.9; 4 rows: 600 15.7 / 16.3, 1000 21.1 / 18.0; 16 rows: 700 17.1 / 20.4, 2304 29.3 / 29.6,
  //   3000 47.6 / 40.8; 32 rows: 700 19.2 / 25.0, 1875 37.0 / 45.9; 64 rows: 1200 51.5 / 64.2, 2304 85.6 / 102; 128 rows: 1000 87.4 / 108
  // Later, with bounds from the last level; rows of a tenth to all of the pages have the same lines (64 rows to 2304: 53.9 / 63.8):
  //   128, 8 heads: 1 row: 1000 17.6 / 16.8; 16 rows: 2304 29.6 / 29.1; 64 rows: 1200 42.4 / 51.8, 2304 62.7 / 73.8
  //   64, 8 heads: 1 row: 600 12.8 / 16.5, 1000 14.7 / 16.6; 16 rows: 2304 23.8 / 25.1; 64 rows: 1200 34.1 / 41.2, 2304 46.3 / 55.5
  //   256, 4 heads: 2 rows: 600 19.7 / 17.8, 1000 25.5 / 18.0; 32 rows: 700 22.5 / 29.0, 2304 46.6 / 41.3; 128 rows: 1200 63.6 / 73.9
  // Heads of 64 would have the lines higher and heads of 256 lower, for a page's bytes: at the lines they lose up to 13% and 18%.
  if (pairs * kSelectThreads<kLarge> > kMostBlocks * kThreads) refuse("too many rows for these heads");
  if (pages <= 640 || (pairs >= 128 && pages <= 2304)) {
    p.how = kLarge;
    return p;
  }
  p.how = kScored;
  p.chunks = (int)((pages + 4 * score_pages_of(b.head_dimension) - 1) / (4 * score_pages_of(b.head_dimension)));
  // The card holds 1024 of these workgroups. With more, each scores little for its start, and a bound far above the rows' own pages leaves many
  // idle: 8 rows of 4000 pages 31.4 us, with 1024 28.3; 32 rows 85.4 and 83.4.
  p.chunks = (int)std::min<uint64_t>(p.chunks, std::max<uint64_t>(1, 1024 / pairs));
  p.stride = (pages + 3) / 4 * 4;
  p.bytes = pairs * p.stride * sizeof(uint32_t);
  return p;
}

void select(int32_t device, void* stream, const hllm_rocm_kv_bounds* bounds, const hllm_rocm_kv_select_args* args) {
  check_bounds(bounds);
  if (!args) refuse("args is null");
  const uint64_t rows = args->rows;
  check_rows(rows);
  if (args->last < 1) refuse("the last page, which may not be whole, is always selected: last is at least 1");
  if ((uint64_t)args->first + args->last > args->keep) refuse("keep is at least first + last");
  if (args->keep > kMostPositions / bounds->page_tokens) refuse("a row of selected pages holds at most 2^30 positions");
  const uint64_t positions = table_positions(args->table_width, args->table_stride, bounds->page_tokens);
  if (rows == 0) return;
  SelectArgs a{};
  a.q = tensor(&args->q, "q", rows, bounds->head_dimension, false);
  if (args->q.heads % bounds->kv_heads) refuse("query heads are a multiple of the cache's heads, at most 1024");
  if (!args->lengths) refuse("lengths is null");
  if (!args->selected || !args->selected_lengths) refuse("selected or selected_lengths is null");
  const SelectPlan plan = plan_select(*bounds, rows, std::min(args->max_length, positions), args->keep);
  if (plan.limit > 0 && !args->page_table) refuse("page_table is null");
  if (plan.bytes > 0 && (!args->workspace || args->workspace_bytes < plan.bytes || (uintptr_t)args->workspace % 16))
    refuse("the workspace is null, not 16-byte aligned or below " + std::to_string(plan.bytes) + " bytes");
  const void* outputs[3] = {args->selected, args->selected_lengths, plan.bytes > 0 ? args->workspace : nullptr};
  const char* names[3] = {"selected", "selected_lengths", "the workspace"};
  for (int i = 0; i < 3; ++i) {
    if (!outputs[i]) continue;
    for (int j = 0; j < i; ++j) check_apart(outputs[i], names[i], outputs[j], names[j]);
    check_apart(outputs[i], names[i], args->page_table, "page_table");
    check_apart(outputs[i], names[i], args->lengths, "lengths");
    check_apart(outputs[i], names[i], args->q.data, "q");
    check_apart(outputs[i], names[i], bounds->codes, "the bounds' codes");
    check_apart(outputs[i], names[i], bounds->scales, "the bounds' scales");
  }
  a.codes = bounds->codes;
  a.scales = bounds->scales;
  a.table = args->page_table;
  a.table_stride = args->table_stride;
  a.lengths = args->lengths;
  a.selected = args->selected;
  a.selected_lengths = args->selected_lengths;
  a.keys = static_cast<uint32_t*>(args->workspace);
  a.stride = plan.stride;
  a.rows = (int32_t)rows;
  a.kv_heads = (int32_t)bounds->kv_heads;
  a.group = (int32_t)(args->q.heads / bounds->kv_heads);
  a.pages = (int32_t)bounds->pages;
  a.page_shift = shift_of(bounds->page_tokens);
  a.limit = (int32_t)plan.limit;
  a.keep = (int32_t)args->keep;
  a.first = (int32_t)args->first;
  a.last = (int32_t)args->last;
  OnDevice on(device);
  launch_select(static_cast<hipStream_t>(stream), args->q.dtype, (int)bounds->head_dimension, plan.how, plan.chunks, a);
  HIP_CHECK(hipGetLastError());
}

}  // namespace
}  // namespace hllm_rocm

// ========================================================================= C ABI

using namespace hllm_rocm;

extern "C" {

hllm_status hllm_rocm_kv_bounds_update(int32_t device, void* stream, const hllm_rocm_kv_pages* pages,
                                       const hllm_rocm_kv_bounds* bounds, const hllm_rocm_kv_bounds_args* args) {
  return guarded([&] {
    check_device(device);
    update_bounds(device, stream, cache_of(pages), bounds, args);
  });
}

hllm_status hllm_rocm_kv4_bounds_update(int32_t device, void* stream, const hllm_rocm_kv4_pages* pages,
                                        const hllm_rocm_kv_bounds* bounds, const hllm_rocm_kv_bounds_args* args) {
  return guarded([&] {
    check_device(device);
    update_bounds(device, stream, cache_of(pages), bounds, args);
  });
}

hllm_status hllm_rocm_kv_select(int32_t device, void* stream, const hllm_rocm_kv_bounds* bounds,
                                const hllm_rocm_kv_select_args* args) {
  return guarded([&] {
    check_device(device);
    select(device, stream, bounds, args);
  });
}

hllm_status hllm_rocm_kv_select_workspace(const hllm_rocm_kv_bounds* bounds, uint64_t rows, uint64_t max_length,
                                          uint32_t keep, uint64_t* bytes) {
  return guarded([&] {
    if (!bytes) refuse("null argument");
    check_bounds(bounds);
    check_rows(rows);
    *bytes = plan_select(*bounds, rows, max_length, keep).bytes;
  });
}

}  // extern "C"
