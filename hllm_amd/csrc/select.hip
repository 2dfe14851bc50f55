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

template <int F, int D>
struct Keys8 {  // eight elements of a position's key as they are held
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
  __device__ void values(float* x) const {
    if constexpr (F < kE2m1) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const floatx4 v = decode4<F>(codes[j]);
#pragma unroll
        for (int i = 0; i < 4; ++i) x[4 * j + i] = v[i] * __uint_as_float(scale);
      }
    } else {
      values8<F>(codes[0], x);
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] *= scale_of<F>(scale);
    }
  }
};

// A value's partner O lanes away in its half, quarter or eighth of the wave, and the value itself, in either order.
template <int O>
__device__ inline float2 both(float v) {
  const uint32_t w = __float_as_uint(v);
  if constexpr (O == 32) {
    const auto x = __builtin_amdgcn_permlane32_swap(w, w, false, false);
    return float2{__uint_as_float(x[0]), __uint_as_float(x[1])};
  } else if constexpr (O == 16) {
    const auto x = __builtin_amdgcn_permlane16_swap(w, w, false, false);
    return float2{__uint_as_float(x[0]), __uint_as_float(x[1])};
  } else {  // a row's lanes go round by O
    return float2{v, __uint_as_float((uint32_t)__builtin_amdgcn_update_dpp(0, (int)w, 0x120 + O, 0xf, 0xf, false))};
  }
}
template <int O>
__device__ inline void widen(float& high, float& low) {
  const float2 h = both<O>(high), l = both<O>(low);
  high = fmaxf(h.x, h.y);
  low = fminf(l.x, l.y);
}

// One wave takes a page and KV head (kWaves = 1), or a workgroup's four share it: a lane has eight channels of every
// (D = 64: eighth, 128: fourth, 256: second) position.
template <int F, int D, int kWaves>
__global__ void __launch_bounds__(kThreads) kv_bounds_kernel(BoundsArgs a) {
  constexpr int L = D / 8, S = 64 / L, kDeep = 4;  // lanes of a vector, positions at once, and of them in flight
  __shared__ float meet[kWaves > 1 ? kWaves : 1][2][kWaves > 1 ? D : 1];
  __shared__ int spoiled[kWaves];
  const Pages& c = a.pages;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const uint64_t item = kWaves > 1 ? blockIdx.x : (uint64_t)blockIdx.x * 4 + wave;
  const int h = (int)(item % c.kv_heads);
  const uint64_t place = item / c.kv_heads;
  const int row = (int)(place / a.places), j = (int)(place - (uint64_t)row * a.places);
  if (row >= a.rows) return;
  const int shift = c.page_shift, length = min(uniform_load(a.lengths + row), a.limit), start = max(uniform_load(a.starts + row), 0);
  const int p = (start >> shift) + j;
  if (start >= length || p > (length - 1) >> shift) return;
  const int id = uniform_load(a.table + (uint64_t)row * a.table_stride + p);
  if (id < 0 || id >= c.pages) return;
  const int count = min(1 << shift, length - (p << shift));
  const int slot = lane / L, d = lane % L * 8;
  const uint64_t page = (uint64_t)id * c.kv_heads + h;
  const uint8_t* from = c.keys + (uint64_t)id * c.page_stride + (uint64_t)h * c.head_stride;
  float high[8], low[8], spoil = 0.0f;
#pragma unroll
  for (int i = 0; i < 8; ++i) high[i] = -INFINITY, low[i] = INFINITY;
  for (int t = kWaves > 1 ? wave * S * kDeep : 0; t < count; t += kWaves * S * kDeep) {
    Keys8<F, D> k[kDeep];
#pragma unroll
    for (int i = 0; i < kDeep; ++i) {
      const int at = min(t + i * S + slot, count - 1);  // the last position again changes nothing
      k[i].load(c, from + (uint64_t)(uint32_t)at * c.token_stride, (page << shift) + at, d);
    }
#pragma unroll
    for (int i = 0; i < kDeep; ++i) {
      float x[8];
      k[i].values(x);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        high[e] = fmaxf(high[e], x[e]);
        low[e] = fminf(low[e], x[e]);
        spoil = fmaf(x[e], 0.0f, spoil);  // NaN once an element is not finite
      }
    }
  }
  bool bad = spoil != 0.0f;  // NaN is not equal
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    if constexpr (L == 8) widen<8>(high[e], low[e]);
    if constexpr (L <= 16) widen<16>(high[e], low[e]);
    widen<32>(high[e], low[e]);
  }
  bad = __any(bad);
  if constexpr (kWaves > 1) {
    if (slot == 0) {
#pragma unroll
      for (int e = 0; e < 8; ++e) meet[wave][0][d + e] = high[e], meet[wave][1][d + e] = low[e];
    }
    if (lane == 0) spoiled[wave] = bad;
    __syncthreads();
    if (wave > 0) return;
#pragma unroll
    for (int w = 1; w < kWaves; ++w) {
      bad |= spoiled[w] != 0;
#pragma unroll
      for (int e = 0; e < 8; ++e) high[e] = fmaxf(high[e], meet[w][0][d + e]), low[e] = fminf(low[e], meet[w][1][d + e]);
    }
  }
  uint32_t most = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) most = max(most, max(__float_as_uint(high[e]) & 0x7fffffffu, __float_as_uint(low[e]) & 0x7fffffffu));
#pragma unroll
  for (int o = 1; o < L; o <<= 1) most = max(most, (uint32_t)__shfl_xor((int)most, o, 64));
  const uint32_t power = whole_power(most);
  const float inverse = __uint_as_float((254u - power) << 23);
  int x[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) x[e] = bad ? 0 : (int)rintf((slot == 0 ? high[e] : low[e]) * inverse);
  if (slot < 2) *reinterpret_cast<uint2v*>(a.codes + (page * 2 + slot) * D + d) = bytes8(x);
  if (lane == 0) a.scales[page] = bad ? NAN : __uint_as_float(power << 23);
}

// ---------------------------------------------------------------- scores

// Numbers' bits so that whole numbers order as the numbers do, -0 as 0; NaN above all of them.
__device__ inline uint32_t ordered(float x) {
  const uint32_t bits = __float_as_uint(x + 0.0f);
  if (x != x) return 0xfffffffeu;
  return bits & 0x80000000u ? ~bits : bits | 0x80000000u;
}

template <int O>
__device__ inline uint32_t row_max(uint32_t v) {
  return max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x120 + O, 0xf, 0xf, false));
}

// The scores of a row's pages for one KV head, as ordered whole numbers: keep(page's place, number). A wave takes sixty-four pages at once,
// from sixty-four `first` on in steps of `step`: with a query's positive and negative elements apart, the sum over channels of the larger product
// is one product [high, low] x [max(q, 0), min(q, 0)] of twice the length, on the matrix units in bytes, with the query heads of a KV
// head as columns. Sums of whole numbers below 2^24 and powers of two are exact.
template <typename T, int D, typename Keep>
__device__ inline void score_pages(const SelectArgs& a, int row, int kvh, int count, int first, int step, Keep&& keep) {
  constexpr int KK = D / 64;
  const int lane = threadIdx.x & 63, quad = lane >> 4, col = lane & 15;
  const int32_t* table = a.table + (uint64_t)row * a.table_stride;
  for (int g0 = 0; g0 < a.group; g0 += 16) {
    const int vectors = min(16, a.group - g0);
    float x[KK][16];
    const T* src = at<const T>(a.q, row, kvh * a.group + g0 + min(col, vectors - 1), 16 * quad);
    uint32_t most = 0;
#pragma unroll
    for (int kk = 0; kk < KK; ++kk) {
      load8(src + 64 * kk, x[kk]);
      load8(src + 64 * kk + 8, x[kk] + 8);
#pragma unroll
      for (int i = 0; i < 16; ++i) most = max(most, __float_as_uint(x[kk][i]) & 0x7fffffffu);
    }
    most = max(most, (uint32_t)__shfl_xor((int)most, 16, 64));
    most = max(most, (uint32_t)__shfl_xor((int)most, 32, 64));
    const bool finite = most < 0x7f800000u;
    const uint32_t power = whole_power(most);
    const float inverse = __uint_as_float((254u - power) << 23), q_scale = finite ? __uint_as_float(power << 23) : NAN;
    int4v up[KK], down[KK];
#pragma unroll
    for (int kk = 0; kk < KK; ++kk)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        int p[8], n[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int v = finite ? (int)rintf(x[kk][8 * i + e] * inverse) : 0;
          p[e] = max(v, 0);
          n[e] = min(v, 0);
        }
        const uint2v pw = bytes8(p), nw = bytes8(n);
        up[kk][2 * i] = (int)pw[0], up[kk][2 * i + 1] = (int)pw[1];
        down[kk][2 * i] = (int)nw[0], down[kk][2 * i + 1] = (int)nw[1];
      }
    // 64 pages at a time, a lane's one of them, whose loads are under way together: in two halves where their bounds take many registers.
    for (int t = 64 * first; t < count; t += 64 * step) {
      const int id = table[min(t + lane, count - 1)];
      const bool there = id >= 0 && id < a.pages;
      const uint64_t absent = __ballot(!there);
      const int own = there ? id : 0;
      const float scale = a.scales[(uint64_t)own * a.kv_heads + kvh];
      constexpr int kTiles = KK < 4 ? 4 : 2;
#pragma unroll
      for (int part = 0; part < 4; part += kTiles) {
        int4v high[kTiles][KK], low[kTiles][KK];
#pragma unroll
        for (int i = 0; i < kTiles; ++i) {
          const uint64_t page = (uint64_t)__shfl(own, 16 * (part + i) + col, 64) * a.kv_heads + kvh;
          const int8_t* from = a.codes + page * (2 * D) + 16 * quad;
#pragma unroll
          for (int kk = 0; kk < KK; ++kk) {
            high[i][kk] = *reinterpret_cast<const int4v*>(from + 64 * kk);
            low[i][kk] = *reinterpret_cast<const int4v*>(from + D + 64 * kk);
          }
        }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = 0; i < kTiles; ++i) {
          int4v dot = {0, 0, 0, 0};
#pragma unroll
          for (int kk = 0; kk < KK; ++kk) {
            dot = __builtin_amdgcn_mfma_i32_16x16x64_i8(high[i][kk], up[kk], dot, 0, 0, 0);
            dot = __builtin_amdgcn_mfma_i32_16x16x64_i8(low[i][kk], down[kk], dot, 0, 0, 0);
          }
          uint32_t mine = 0;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int of = 16 * (part + i) + 4 * quad + e;
            const float by = __shfl(scale, of, 64);
            uint32_t v = col < vectors ? ordered((float)dot[e] * by * q_scale) : 0u;
            v = row_max<1>(row_max<2>(row_max<4>(row_max<8>(v))));
            if (absent >> of & 1) v = 0;
            if (col == e) mine = v;
          }
          const int place = t + 16 * (part + i) + 4 * quad + col;
          if (col < 4 && place < count) keep(place, mine, g0 > 0);
        }
      }
    }
  }
}

__device__ inline int pages_of(const SelectArgs& a, int row, int& length) {
  length = min(uniform_load(a.lengths + row), a.limit);
  return length <= 0 ? 0 : ((length - 1) >> a.page_shift) + 1;
}

// Scores into the workspace, for rows of more pages than one workgroup scores.
template <typename T, int D>
__global__ void __launch_bounds__(kThreads) kv_score_kernel(SelectArgs a) {
  const int row = blockIdx.x / a.kv_heads, kvh = blockIdx.x % a.kv_heads;
  int length;
  const int count = pages_of(a, row, length);
  if (count <= a.keep) return;
  uint32_t* keys = a.keys + (uint64_t)blockIdx.x * a.stride;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  score_pages<T, D>(a, row, kvh, count, blockIdx.y * 4 + wave, gridDim.y * 4,
                    [&](int place, uint32_t key, bool again) { keys[place] = again ? max(keys[place], key) : key; });
}

// ---------------------------------------------------------------- selection

constexpr int kOwn = 16;  // scores that a thread holds

// A workgroup selects a row's pages for one KV head: it finds, from the upper bit down, the largest number that `keep` scores
// reach, then writes the pages above it, and of those at it the first ones, in their order. kHere: it has scored
// them itself (at most kThreads * kOwn).
template <typename T, int D, bool kHere>
__global__ void __launch_bounds__(kThreads) kv_select_kernel(SelectArgs a) {
  __shared__ uint32_t scored[kHere ? kThreads * kOwn : 1];
  __shared__ uint32_t range[4][2];
  __shared__ int counts[2][4];
  __shared__ int before[kOwn][4][2];
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
    for (int i = threadIdx.x; i < a.keep; i += kThreads) out[i] = i < n ? table[i] : -1;
    return;
  }
  const uint32_t* keys = a.keys + (uint64_t)blockIdx.x * a.stride;
  if constexpr (kHere) {
    score_pages<T, D>(a, row, kvh, n, wave, 4,
                      [&](int place, uint32_t key, bool again) { scored[place] = again ? max(scored[place], key) : key; });
    __syncthreads();
  }
  const int tiles = kHere ? 1 : (n + kThreads * kOwn - 1) / (kThreads * kOwn);
  uint32_t v[kOwn];
  int used = 0;  // of v, the same for all threads
  const auto load = [&](int tile) {
    const int from = tile * kThreads * kOwn;
    used = min(kOwn, (n - from + kThreads - 1) / kThreads);
#pragma unroll
    for (int j = 0; j < kOwn; ++j) {
      const int i = from + j * kThreads + (int)threadIdx.x;
      v[j] = 0;
      if (i < n) v[j] = i < a.first || i >= n - a.last ? 0xffffffffu : kHere ? scored[i] : keys[i];
    }
  };
  load(0);
  // Bits that all scores share are the threshold's. Places behind the last page are left out; forced ones have every bit.
  uint32_t all = 0xffffffffu, some = 0;
  for (int tile = 0; tile < tiles; ++tile) {
    if (tile > 0) load(tile);
#pragma unroll
    for (int j = 0; j < kOwn; ++j) {
      const int i = tile * kThreads * kOwn + j * kThreads + (int)threadIdx.x;
      if (i < n && i >= a.first && i < n - a.last) all &= v[j], some |= v[j];
    }
  }
  for (int o = 1; o < 64; o <<= 1) {
    all &= (uint32_t)__shfl_xor((int)all, o, 64);
    some |= (uint32_t)__shfl_xor((int)some, o, 64);
  }
  if (lane == 0) range[wave][0] = all, range[wave][1] = some;
  __syncthreads();
  all = range[0][0] & range[1][0] & range[2][0] & range[3][0];
  some = range[0][1] | range[1][1] | range[2][1] | range[3][1];
  // keep > first + last: some score is selected by its number, and the threshold is one of theirs.
  const int forced = a.first + a.last;
  uint32_t threshold = 0xffffffffu;
  int above = forced;   // scores that are larger than the threshold
  bool whole = a.keep == forced;   // the threshold's own scores are all selected
  if (!whole) {
    const int bits = all == some ? 0 : 32 - __builtin_clz(all ^ some);
    threshold = bits == 32 ? 0 : all >> bits << bits;
    for (int b = bits - 1; b >= 0 && !whole; --b) {
      const uint32_t next = threshold | 1u << b;
      int reach = 0;
      for (int tile = 0; tile < tiles; ++tile) {
        if (tiles > 1) load(tile);
#pragma unroll
        for (int j = 0; j < kOwn; ++j)
          if (j < used) reach += __popcll(__ballot(v[j] >= next));
      }
      if (lane == 0) counts[b & 1][wave] = reach;
      __syncthreads();
      reach = counts[b & 1][0] + counts[b & 1][1] + counts[b & 1][2] + counts[b & 1][3];
      if (reach >= a.keep) threshold = next;
      whole = reach == a.keep;
    }
  }
  // Places in order: first by v's index, then by wave and lane.
  int larger = 0, equal = 0;  // of the tiles before, and of this tile's places before the thread's
  const uint64_t below = (1ull << lane) - 1;
  if (!whole) {
    above = 0;
    for (int tile = 0; tile < tiles; ++tile) {
      if (tiles > 1) load(tile);
#pragma unroll
      for (int j = 0; j < kOwn; ++j)
        if (j < used) above += __popcll(__ballot(v[j] > threshold));
    }
    __syncthreads();
    if (lane == 0) counts[0][wave] = above;
    __syncthreads();
    above = counts[0][0] + counts[0][1] + counts[0][2] + counts[0][3];
  }
  const int take = whole ? 0x7fffffff : a.keep - above;  // of the threshold's own scores
  for (int tile = 0; tile < tiles; ++tile) {
    if (tiles > 1) load(tile);
    if (tile > 0) __syncthreads();
#pragma unroll
    for (int j = 0; j < kOwn; ++j) {
      if (j >= used) continue;
      const int i = tile * kThreads * kOwn + j * kThreads + (int)threadIdx.x;
      const int g = __popcll(__ballot(i < n && v[j] > threshold)), e = __popcll(__ballot(i < n && v[j] == threshold));
      if (lane == 0) before[j][wave][0] = g, before[j][wave][1] = e;
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < kOwn; ++j) {
      if (j >= used) continue;
      const int i = tile * kThreads * kOwn + j * kThreads + (int)threadIdx.x;
      const bool gt = i < n && v[j] > threshold, eq = i < n && v[j] == threshold;
      int g = larger, e = equal;
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        if (w < wave) g += before[j][w][0], e += before[j][w][1];
        larger += before[j][w][0], equal += before[j][w][1];
      }
      g += __popcll(__ballot(gt) & below);
      e += __popcll(__ballot(eq) & below);
      if (gt || (eq && e < take)) out[g + min(e, take)] = table[i];
    }
  }
}

template <int F>
void bounds_format(hipStream_t stream, int head_dim, const BoundsArgs& a) {
  const uint64_t items = (uint64_t)a.rows * a.places * a.pages.kv_heads;
  const auto run = [&](auto dim) {
    constexpr int D = decltype(dim)::value;
    if (a.wide)
      kv_bounds_kernel<F, D, 4><<<(unsigned)items, kThreads, 0, stream>>>(a);
    else
      kv_bounds_kernel<F, D, 1><<<(unsigned)((items + 3) / 4), kThreads, 0, stream>>>(a);
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
void select_dim(hipStream_t stream, int chunks, const SelectArgs& a) {
  const unsigned pairs = (unsigned)(a.rows * a.kv_heads);
  if (chunks == 0) {
    kv_select_kernel<T, D, true><<<pairs, kThreads, 0, stream>>>(a);
  } else {
    kv_score_kernel<T, D><<<dim3(pairs, chunks), kThreads, 0, stream>>>(a);
    kv_select_kernel<T, D, false><<<pairs, kThreads, 0, stream>>>(a);
  }
}

void launch_select(hipStream_t stream, uint32_t dtype, int head_dim, int chunks, const SelectArgs& a) {
  const auto run = [&](auto zero) {
    using T = decltype(zero);
    if (head_dim == 64) select_dim<T, 64>(stream, chunks, a);
    if (head_dim == 128) select_dim<T, 128>(stream, chunks, a);
    if (head_dim == 256) select_dim<T, 256>(stream, chunks, a);
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
  a.wide = cache.page_tokens > 128;
  OnDevice on(device);
  launch_bounds(static_cast<hipStream_t>(stream), cache.format, cache.head_dim, a);
  HIP_CHECK(hipGetLastError());
}

// Pages that the workgroup that selects scores itself at most: 64 for each of its waves, twice.
constexpr uint64_t kHerePages = 512;

// How a selection's rows are scored: `chunks` workgroups a row and KV head before the one that selects, 0: by that one.
struct SelectPlan {
  uint64_t limit = 0, stride = 0, bytes = 0;
  int chunks = 0;
};

SelectPlan plan_select(const hllm_rocm_kv_bounds& b, uint64_t rows, uint64_t max_length, uint64_t keep) {
  SelectPlan p;
  p.limit = std::min(max_length, kMostPositions);
  const uint64_t pages = (p.limit + b.page_tokens - 1) / b.page_tokens, pairs = rows * b.kv_heads;
  if (pairs > kMostBlocks) refuse("too many rows for these heads");
  if (rows == 0 || pages <= keep) return p;
  if (pages <= kHerePages) return p;
  p.chunks = (int)((pages + 255) / 256);  // a wave scores 64 pages
  if (pairs * p.chunks > kMostBlocks) p.chunks = (int)(kMostBlocks / pairs);
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
  launch_select(static_cast<hipStream_t>(stream), args->q.dtype, (int)bounds->head_dimension, plan.chunks, a);
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
