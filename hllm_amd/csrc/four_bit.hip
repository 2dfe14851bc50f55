// Kernels over the 4-bit paged cache: its vectors read back, and one new token's attention over it. (Rows are written by
// the rotation's kernel.)
#include <algorithm>
#include <atomic>

#include "operators_device.hpp"

namespace hllm_rocm {
namespace {

// ---------------------------------------------------------------- codes

// Eight E2M1 codes of a word times their group's power of two, as BF16.
__device__ inline bhalf8 scaled8(uint32_t w, float scale) {
  const auto a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 0), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 1),
             c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 2), d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 3);
  return bhalf8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// Eight INT4 codes of a word as F16, which holds every code exactly; code i lies beside i + 4.
__device__ inline half8 halves8(uint32_t w) {
  const half2v a = low_halves(w), b = high_halves(w), c = low_halves(w >> 8), d = high_halves(w >> 8);
  return half8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// The scale of group g among a position's.
template <int F>
__device__ inline float held_scale(const uint32_t* raw, int g) {
  return scale_of<F>(F == kE2m1 ? raw[g / 4] >> (8 * (g % 4)) & 255u : raw[g / 2] >> (16 * (g % 2)) & 0xffffu);
}

// ---------------------------------------------------------------- reading back

// A thread reads the codes of sixteen bytes of output of a key, and of the value beside it, and writes them. A value's
// codes lie G bytes apart (two elements of each group beside each other). Nothing but memory traffic, nearly all of it written:
// 30000 positions of 8 heads of 128 to F16 33.4 us, 4.7 TB/s (a copy of 2 GiB reaches 4.9).
template <typename T, int F, int D>
__global__ void __launch_bounds__(kThreads) kv4_read_kernel(ReadArgs a) {
  constexpr int kCodes = 16 / sizeof(T), L = D / kCodes, G = D / 32;
  const Pages& c = a.pages;
  const uint32_t per_row = (uint32_t)c.kv_heads * L;
  const uint64_t unit = (uint64_t)blockIdx.x * kThreads + threadIdx.x;
  const uint64_t row = unit / per_row;
  if (row >= (uint64_t)a.rows) return;
  const int in_row = (int)(unit - row * per_row), h = in_row / L, d = in_row % L * kCodes, g = d / 32;
  const int slot = a.slots[row];
  if (slot < 0 || (slot >> c.page_shift) >= c.pages) return;
  const int page = slot >> c.page_shift, offset = slot & ((1 << c.page_shift) - 1);
  const uint64_t from = (uint64_t)page * c.page_stride + (uint64_t)offset * c.token_stride + (uint64_t)h * c.head_stride;
  const uint64_t scale_at = ((((uint64_t)page * c.kv_heads + h) << c.page_shift) + offset) * G + g;
  uint32_t codes[2] = {0, 0};
  if constexpr (kCodes == 8) {
    codes[0] = *reinterpret_cast<const uint32_t*>(c.keys + from + d / 2);
    // A vector's lanes read a word each and take the bytes of their eight elements from one another.
    const uint32_t word = *reinterpret_cast<const uint32_t*>(c.values + from + d / 2);
    const int lane = threadIdx.x & 63, base = lane & ~(L - 1);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int at = G * (d % 32 / 2 + i) + g;
      codes[1] |= ((uint32_t)__shfl((int)word, base + at / 4, 64) >> (8 * (at % 4)) & 255u) << (8 * i);
    }
  } else {
    codes[0] = *reinterpret_cast<const uint16_t*>(c.keys + from + d / 2);
#pragma unroll
    for (int i = 0; i < 2; ++i) codes[1] |= (uint32_t)c.values[from + G * (d % 32 / 2 + i) + g] << (8 * i);
  }
  float scale[2];
  if constexpr (F == kE2m1) {
    scale[0] = scale_of<F>(static_cast<const uint8_t*>(c.key_scales)[scale_at]);
    scale[1] = scale_of<F>(static_cast<const uint8_t*>(c.value_scales)[scale_at]);
  } else {
    scale[0] = scale_of<F>(static_cast<const uint16_t*>(c.key_scales)[scale_at]);
    scale[1] = scale_of<F>(static_cast<const uint16_t*>(c.value_scales)[scale_at]);
  }
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    T* to = at<T>(which ? a.v : a.k, (int)row, h, d);
    float x[8];
    values8<F>(codes[which], x);
    if constexpr (kCodes == 8) {
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] *= scale[which];
      store8(to, x);
    } else {
      store4(to, floatx4{x[0], x[1], x[2], x[3]} * scale[which]);
    }
  }
}

// ---------------------------------------------------------------- attention

// A wave's tile of N positions in LDS: the codes of keys and of values, then their scales. A position lies in slot `slot` and a
// row's sixteen-byte chunks are permuted (chunk k at k ^ swizzle), so that the rows that are read at once, of
// four eights of positions, lie in different banks, keys and values alike. The keys' scales are kept as they are held (E2M1),
// or as F32 numbers, each group's N together (INT4). The values' are too: as ratios to a power of two near the largest
// of the position's, in F16 (16-bit tensors), or as themselves in F32; and that power, or the largest, for each position.
template <typename T, int F, int D>
struct Tile4 {
  static constexpr int N = kAttend4Tile<D>, kRow = D / 2, kChunks = kRow / 16, G = D / 32;
  static constexpr bool kRatios = sizeof(T) == 2;
  static constexpr int kCodes = N * kRow, kScales = 4 * kCodes, kValueScales = kScales + G * N * 4;
  static constexpr int kLargest = kValueScales + G * N * (kRatios ? 2 : 4);
  static constexpr int kBytes = (std::max(kLargest + N * 4, 64 * D) + 255) / 256 * 256, kBlock = kThreads / 64 * kBytes;
  static constexpr int kGroups = N / 8;   // eights of positions, each in one page
  static constexpr int kCopies = kCodes / 1024;
  static constexpr int kHalf = 4 * kRow;  // from a slot of the first thirty-two positions to that of the next
  static __device__ int slot(int eight, int offset) {
    return offset * kGroups + (D == 64 ? eight ^ (offset >> 1 & 1) << 2 : eight);
  }
  static __device__ int swizzle(int eight, int offset) {
    return D == 64 ? offset & 1 : D == 128 ? offset & 3 : (offset & 3) | (eight >> 1) << 2;
  }
  // Byte `b` of the row of one of the first thirty-two positions, or of the one `half` = kHalf s bytes on.
  static __device__ int at(int eight, int offset, int b, int half) {
    const int first = slot(eight, offset) * kRow + ((b / 16 ^ swizzle(eight, offset)) * 16) + b % 16;
    return D == 64 ? first ^ half : first + half;
  }
};

// Which pair or share a workgroup takes. The workgroups of a cluster, whose pairs read the same cache lines, take the same share of
// each of them, at once and on the same of the card's eight dies, round which workgroups go and which have a cache each.
__device__ inline int place_of(const AttendArgs& a, int block) {
  const int die = block & 7, i = block >> 3;
  return ((i / a.cluster) * 8 + die) * a.cluster + i % a.cluster;
}

// As kv_attention_kernel (operators.hip): a pair's scores S = K Q^T and sums O^T = V^T P are products on the matrix units,
// with the softmax's sum in F32. What differs comes from the scales that 32 elements of a vector share. E2M1 keys become BF16 with
// their scale, which holds them exactly (queries as one to three BF16 parts); INT4 keys enter as F16 numbers, and the sums of
// each group's 16 x 16 x 32 product are multiplied by its scale in F32. A value's scales enter the weights, which are made for each
// group by itself, so values enter as codes. A key's codes lie in order: a lane's word is eight elements of one group. A value's
// codes lie so that a lane's bytes of a position are two elements of each group: the sixteen rows of an output fragment have one group.
//
// Bound by the cache's bytes where it is long and heads lie apart: 24 rows of 12000 to 30000 positions, 32 / 8 heads of 128, E2M1, BF16
// 101 us, 5.1 TB/s (a streaming read 6.3); INT4, whose scales take a product of their own each, 125 us, 4.3 TB/s; F32, with two
// or three times the products, 149. Two tiles a wave in LDS, so that one is under way while the other is worked on: 12 waves a CU have 52 KB
// in flight. Heads within a cache line, read as clusters, 121 us. Short rows are a chain of start, page, tile and join: 64 rows to
// 2048 positions 22 us. The native product of E2M1 codes with scales
// was measured to err by up to 2^-13 of its sum of magnitudes and is not used.
template <typename T, int F, int D>
__global__ void __launch_bounds__(kThreads, kAttend4Blocks<D>) kv4_attention_kernel(AttendArgs a) {
  using Layout = Tile4<T, F, D>;
  constexpr int N = Layout::N, G = Layout::G, H = N / 32, kStep = 4 * N;
  constexpr int W = (G + 3) / 4;             // words of a lane's value bytes of a position
  constexpr int SB = F == kE2m1 ? G : 2 * G; // scale bytes of a position
  constexpr int P = sizeof(T) == 4 ? 2 : 1;  // F16 parts of a weight
  using Query = std::conditional_t<F == kE2m1, bhalf, _Float16>;
  constexpr int Q = F == kInt4 ? P : sizeof(T) == 4 ? 3 : std::is_same_v<T, bhalf> ? 1 : 2;  // parts of a query element
  typedef Query query8 __attribute__((ext_vector_type(8)));
  constexpr bool kRatios = Layout::kRatios;
  constexpr bool kBoth = N == 32;            // a lane holds a position's key or value scales, not both
  extern __shared__ __attribute__((aligned(256))) char smem[];
  __shared__ float states[4][3][16];
  __shared__ query8 queries[Q][G][64];

  const Pages& c = a.pages;
  const int KVH = c.kv_heads, shift = c.page_shift, in_row = KVH * a.head_groups;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int quad = lane >> 4, col = lane & 15;
  const int place = place_of(a, blockIdx.x);
  if (place >= a.blocks) return;
  // Shares are counted in clusters.
  const int cluster = a.cluster, me = place / cluster, member = place - me * cluster;
  Share<kStep, kPair4Cost> share;
  if (!share.first_pair(a, in_row / cluster, me, a.blocks / cluster, lane)) return;

  bool again = false;
  for (bool more = true; more; more = share.next_pair(a, in_row / cluster)) {
  const int row = share.row, kvg = share.kvg * cluster + member, length = share.length;
  // This share's steps of the pair, low .. high - 1, and the workgroups that have others.
  const int steps = steps_of<kStep>(length), first_unit = share.start + kPair4Cost;
  const int low = max(share.from - first_unit, 0), high = min(steps, share.to - first_unit);
  if (steps > 0 ? low >= high : share.start < share.from) continue;  // only the cost of starting it is this share's
  const int first = first_unit / share.budget;
  const int parts = a.shared && steps > 0 ? (first_unit + steps - 1) / share.budget - first + 1 : 1;
  const int kvh = kvg / a.head_groups, g0 = (kvg - kvh * a.head_groups) * 16;
  const int begin = kStep * low, end = min(length, kStep * high);
  if (again) __syncthreads();  // the workgroup has read the last pair's sums
  again = true;
  const int vectors = min(16, a.group - g0);

  const int32_t* table = a.table + (uint64_t)row * a.table_stride + (uint64_t)kvh * a.table_head;
  const int mask = (1 << shift) - 1;
  const uint32_t token = c.token_stride;
  char* tile = smem + wave * Layout::kBytes;
  const uint32_t tile_at = (uint32_t)(size_t)((__attribute__((address_space(3))) char*)smem) + wave * Layout::kBytes;

  // A lane's share of the copies: chunks of the positions `offset` (+ a step for each copy) of one eight. Copy i's
  // first lane has slot 64 i / kChunks.
  constexpr int kPer = 64 / Layout::kChunks;  // slots of a copy
  const int s0 = lane / Layout::kChunks, offset0 = s0 / Layout::kGroups;
  const int eight = s0 % Layout::kGroups ^ (D == 64 ? (offset0 >> 1 & 1) << 2 : 0);
  constexpr int kOffsets = kPer / Layout::kGroups;  // 2 or 4 positions of each eight
  const uint8_t* keys = c.keys + (uint64_t)kvh * c.head_stride + (uint64_t)offset0 * token;
  const uint64_t values_at = (uint64_t)(c.values - c.keys);
  // Its scales: of position lane (N = 64), or of position lane % 32, the keys' or the values'.
  const int own = lane & (N - 1);
  const uint8_t* scales = static_cast<const uint8_t*>(kBoth && lane >= 32 ? c.value_scales : c.key_scales);
  const uint64_t value_scales_at = static_cast<const uint8_t*>(c.value_scales) - static_cast<const uint8_t*>(c.key_scales);

  // The page of the lane's scales' position (of the last position's page behind the part).
  const auto page_of = [&](int t) { return table[min(t + (own & ~7), end - 1) >> shift]; };
  uint32_t held[2][SB > 4 ? SB / 4 : 1];  // scales as they are held, of the next tile
  const auto load_scales = [&](uint32_t* to, const uint8_t* from) {
    if constexpr (SB == 2) to[0] = *reinterpret_cast<const uint16_t*>(from);
    if constexpr (SB == 4) to[0] = *reinterpret_cast<const uint32_t*>(from);
    if constexpr (SB == 8) {
      const uint2v w = *reinterpret_cast<const uint2v*>(from);
      to[0] = w[0], to[1] = w[1];
    }
    if constexpr (SB == 16) {
      const uint4v w = *reinterpret_cast<const uint4v*>(from);
#pragma unroll
      for (int i = 0; i < 4; ++i) to[i] = w[i];
    }
  };
  // Starts a tile's copies and loads its scales; returns a bit for each eight whose page is not there.
  const auto copy_tile = [&](int t, int id, int buffer) {
    const bool there = id >= 0 && id < c.pages;
    const uint64_t absent = __ballot(!there);
    const int page = there ? id : 0;
    const int from_page = __shfl(page, eight * 8, 64);
    const uint8_t* from = keys + (uint64_t)(uint32_t)from_page * c.page_stride + (uint64_t)(uint32_t)((t + 8 * eight) & mask) * token;
#pragma unroll
    for (int i = 0; i < Layout::kCopies; ++i) {
      const int chunk = (lane % Layout::kChunks) ^ Layout::swizzle(eight, offset0 + i * kOffsets);
      const uint8_t* at = from + (uint64_t)(i * kOffsets) * token + chunk * 16;
      if (cluster > 1) {  // others read the lines' rest; lines that are read once are not kept (head-major, long: 97 us, not 103)
        lds_copy16_at(at, tile_at + buffer + i * 1024);
        lds_copy16_at(at + values_at, tile_at + buffer + Layout::kCodes + i * 1024);
      } else {
        lds_stream16_at(at, tile_at + buffer + i * 1024);
        lds_stream16_at(at + values_at, tile_at + buffer + Layout::kCodes + i * 1024);
      }
    }
    const uint8_t* at = scales + ((((uint64_t)page * KVH + kvh) << shift) + ((t + own) & mask)) * SB;
    load_scales(held[0], at);
    if constexpr (!kBoth) load_scales(held[1], at + value_scales_at);
    int missing = 0;
#pragma unroll
    for (int e = 0; e < Layout::kGroups; ++e) missing |= (int)(absent >> (8 * e) & 1) << e;
    return missing;
  };

  int t = begin + N * wave, missing = 0, id = 0;
  if (t < end) {
    missing = copy_tile(t, page_of(t), 0);
    id = page_of(min(t + kStep, end - 1));
  }

  // Q^T as the B operand, kept in LDS for the four waves: group g's lane (col, quad) holds elements 32 g + 8 quad + j in the order of
  // halves8. Each vector is divided by the power of two of its largest element, which puts F32 and BF16
  // ranges into F16's and goes back into its scores. E2M1 keys take it as one to three BF16 numbers, its eight, eleven or 24 bits.
  float factor, factor_lo;
  {
    float x[G][8];
    const T* src = at<const T>(a.q, row, kvh * a.group + g0 + min(col, vectors - 1), 8 * quad);
    uint32_t most = 0;
#pragma unroll
    for (int g = 0; g < G; ++g) {
      load8(src + 32 * g, x[g]);
#pragma unroll
      for (int j = 0; j < 8; ++j) most = max(most, __float_as_uint(x[g][j]) & 0x7fffffffu);
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
      for (int g = 0; g < G; ++g) {
        query8 part[Q];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          float y = x[g][F == kE2m1 ? j : (j >> 1) + 4 * (j & 1)] * down;
#pragma unroll
          for (int p = 0; p < Q; ++p) {
            part[p][j] = (Query)y;
            y -= (float)part[p][j];
          }
        }
#pragma unroll
        for (int p = 0; p < Q; ++p) queries[p][g][lane] = part[p];
      }
    }
  }
  __syncthreads();

  // Where they are few, in registers.
  constexpr bool kHeld = Q * G <= 4;
  query8 held_q[kHeld ? Q : 1][kHeld ? G : 1];
  if constexpr (kHeld) {
#pragma unroll
    for (int g = 0; g < G; ++g)
#pragma unroll
      for (int p = 0; p < Q; ++p) held_q[p][g] = queries[p][g][lane];
  }

  // Weights, their scaling by r and the sums o as in kv_attention_kernel, r by each position's largest value scale.
  // o[2 g + e]'s row c is element 32 g + 2 c + e.
  floatx4 o[2 * G];
#pragma unroll
  for (int f = 0; f < 2 * G; ++f) o[f] = floatx4{0.f, 0.f, 0.f, 0.f};
  float m = -INFINITY, l = 0.0f, r = 0.0f;
  // A position whose values are all 0 has a scale that no other has; kLeast: what counts as its power of two.
  constexpr int kNoUnit = -1000, kNoScale = 1, kLeast = -190;
  int unit = kNoUnit;  // 16-bit tensors: the exponent of the value scales' unit
  const auto largest_of = [](int v) { return __builtin_amdgcn_readfirstlane((int)wave_max((uint32_t)v)); };
  // A reference that takes an exponent is rounded by 2^-24 of itself, like a score; past 2^12 they are whole numbers, which F32 adds exactly,
  // and past 2^23, where it does not, they stay where they are.
  const auto moves = [&] { return fabsf(m) < 0x1p23f || m == -INFINITY; };
  // Another unit for the value scales, 2^by as large: the columns' references come down by as much, or their sums of values do.
  const auto move_unit = [&](int by) {
    const int step = moves() ? by : 0;
    const float rest = __builtin_amdgcn_ldexpf(1.0f, step - by);
#pragma unroll
    for (int f = 0; f < 2 * G; ++f) o[f] *= rest;
    l = __builtin_amdgcn_ldexpf(l, step);
    m -= (float)step;
    unit += by;
  };
  bool any = false;  // whether the wave has had a position
  float* key_scale = reinterpret_cast<float*>(tile + Layout::kScales);
  char* value_scale = tile + Layout::kValueScales;
  float* largest_scale = reinterpret_cast<float*>(tile + Layout::kLargest);

  int buffer = 0;
  for (; t < end; t += kStep) {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    const int gone = missing;
    const bool whole = gone == 0 && t + N <= end;
    any |= gone != (1 << Layout::kGroups) - 1;  // eights behind the end count as the last one's page
    {
      // The lane's scales. Values past the part and in pages that are not there have none.
      const bool counts = whole || (t + own < end && !(gone >> (own >> 3) & 1));
      const auto keep_keys = [&](const uint32_t* raw) {
        if constexpr (F == kE2m1) {
          float v[G];
#pragma unroll
          for (int g = 0; g < G; ++g) v[g] = __uint_as_float((raw[g / 4] >> (8 * (g % 4)) & 255u) << 23);
          if constexpr (G == 2) *reinterpret_cast<float2*>(key_scale + G * own) = float2{v[0], v[1]};
#pragma unroll
          for (int g = 0; g + 3 < G; g += 4) *reinterpret_cast<floatx4*>(key_scale + G * own + g) = floatx4{v[g], v[g + 1], v[g + 2], v[g + 3]};
        } else {
#pragma unroll
          for (int g = 0; g < G; ++g) key_scale[g * N + own] = held_scale<F>(raw, g);
        }
      };
      const auto keep_values = [&](const uint32_t* raw, bool mine) {
        float v[G], most = 0.0f;
#pragma unroll
        for (int g = 0; g < G; ++g) {
          v[g] = counts ? held_scale<F>(raw, g) : 0.0f;
          most = fmaxf(most, fabsf(v[g]));  // NaN is not taken
        }
        if constexpr (kRatios) {
          const bool some = mine && most > 0.0f;
          const int power = max((int)(__float_as_uint(most) >> 23), 1);
          if (__any(some && (uint32_t)(power - unit + 125) > 133u)) {
            const int top = largest_of(some ? power : 0);
            // Up as far as the sums of weights leave room for it, to the largest; down to what F32 holds beside the smallest.
            if (unit == kNoUnit) unit = top;
            int by = 0;
            if (top > unit + 8) {
              const int sums = largest_of(l < INFINITY && moves() ? (int)(__float_as_uint(l) >> 23) : 0);
              by = min(top - unit, max(226 - sums, 0));
            }
            if (__any(some && power < unit + by - 125)) {
              const int least = 255 - largest_of(some ? 255 - power : 0);
              by = min(by, max(least + 125, top - 120) - unit);
            }
            if (by != 0) move_unit(by);
          }
          if (mine) {
            const int held = some ? min(max(power - unit + 127, kNoScale), 254) : unit == kNoUnit ? 127 : kNoScale;
            largest_scale[own] = __uint_as_float((uint32_t)held << 23);
#pragma unroll
            for (int g = 0; g < G; ++g)
              reinterpret_cast<_Float16*>(value_scale)[g * N + own] = (_Float16)__builtin_amdgcn_ldexpf(v[g], 127 - power);
          }
        } else if (mine) {
          largest_scale[own] = most;
#pragma unroll
          for (int g = 0; g < G; ++g) reinterpret_cast<float*>(value_scale)[g * N + own] = v[g];
        }
      };
      if (!kBoth || lane < 32) keep_keys(held[0]);
      keep_values(held[kBoth ? 0 : 1], !kBoth || lane >= 32);
    }
    const char* codes = tile + buffer;
    const auto next_tile = [&] {
      if (t + kStep < end) {
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        buffer = 2 * Layout::kCodes - buffer;
        missing = copy_tile(t + kStep, id, buffer);
        id = page_of(min(t + 2 * kStep, end - 1));
      }
    };
    next_tile();
    // The tile's positions in thirty-twos, one after the other.
#pragma unroll 1
    for (int s = 0; s < H; ++s) {
      // Score fragment h's row 4 q + i is position 8 q + 4 h + i: a lane's scores are positions 8 quad .. + 7, which are
      // also its slots of the value products.
      const int half = s * Layout::kHalf;
      // What a product needs is read from LDS well before it: a read takes as long as some thirty instructions.
      uint32_t kw[G][2];
      query8 q[kHeld ? 1 : Q][kHeld ? 1 : G];
#pragma unroll
      for (int g = 0; g < G; ++g) {
#pragma unroll
        for (int h = 0; h < 2; ++h)
          kw[g][h] = *reinterpret_cast<const uint32_t*>(codes + Layout::at(col >> 2, 4 * h + (col & 3), 16 * g + 4 * quad, half));
        if constexpr (!kHeld) {
#pragma unroll
          for (int p = 0; p < Q; ++p) q[p][g] = queries[p][g][lane];
        }
      }
      const auto query = [&](int p, int g) { return kHeld ? held_q[kHeld ? p : 0][kHeld ? g : 0] : q[kHeld ? 0 : p][kHeld ? 0 : g]; };
      float d[8];
      if constexpr (F == kE2m1) {
        // A key's elements as BF16, which holds every code times its scale exactly.
        floatx4 x[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
        float by[2][G];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const float* at = key_scale + G * (32 * s + 8 * (col >> 2) + 4 * h + (col & 3));
          if constexpr (G == 2) {
            const float2 w = *reinterpret_cast<const float2*>(at);
            by[h][0] = w.x, by[h][1] = w.y;
          }
#pragma unroll
          for (int g = 0; g + 3 < G; g += 4) {
            const floatx4 w = *reinterpret_cast<const floatx4*>(at + g);
#pragma unroll
            for (int i = 0; i < 4; ++i) by[h][g + i] = w[i];
          }
        }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int g = 0; g < G; ++g)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const bhalf8 k = scaled8(kw[g][h], by[h][g]);
#pragma unroll
            for (int p = Q - 1; p >= 0; --p) x[h] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k, query(p, g), x[h], 0, 0, 0);
          }
#pragma unroll
        for (int j = 0; j < 8; ++j) d[j] = x[j >> 2][j & 3];
      } else {
        floatx4 by[G][2];
#pragma unroll
        for (int g = 0; g < G; ++g)
#pragma unroll
          for (int h = 0; h < 2; ++h) by[g][h] = *reinterpret_cast<const floatx4*>(key_scale + g * N + 32 * s + 8 * quad + 4 * h);
        if constexpr (G <= 4) __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int j = 0; j < 8; ++j) d[j] = 0.0f;
#pragma unroll
        for (int g = 0; g < G; ++g)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const half8 k = halves8(kw[g][h]);
            floatx4 x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int p = Q - 1; p >= 0; --p) x = mfma(k, query(p, g), x);
#pragma unroll
            for (int i = 0; i < 4; ++i) d[4 * h + i] = fmaf(x[i], by[g][h][i], d[4 * h + i]);
          }
      }
      uint32_t vw[8][W];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const char* line = codes + Layout::kCodes + Layout::at(quad, j, G * col, half);
        if constexpr (G == 2) vw[j][0] = *reinterpret_cast<const uint16_t*>(line);
        if constexpr (G == 4) vw[j][0] = *reinterpret_cast<const uint32_t*>(line);
        if constexpr (G == 8) {
          const uint2v w = *reinterpret_cast<const uint2v*>(line);
          vw[j][0] = w[0];
          vw[j][1] = w[1];
        }
      }
      const int valid = whole ? 8 : gone >> (4 * s + quad) & 1 ? 0 : end - (t + 32 * s + 8 * quad);
      float weight[8], ls[8];
      half8 ratio_weight, ratios[kRatios ? G : 1];
      load8(largest_scale + 32 * s + 8 * quad, ls);
      if constexpr (kRatios) {
#pragma unroll
        for (int g = 0; g < G; ++g) ratios[g] = *reinterpret_cast<const half8*>(value_scale + 2 * (g * N + 32 * s + 8 * quad));
        __builtin_amdgcn_sched_barrier(0);
      }
      if constexpr (kRatios) {
        // Weights are 2^(score - m) for an m that is seldom changed: where a wave's first scores are found, and where a weight times its
        // value scales (in `unit`s) is above 2^14, or a weight above 2^100; the largest is then made 2^6. So most
        // tiles need no maximum, and F16 holds every weight to 2^-11 or to 2^-31 of the largest. Where a weight would have to be above 2^100
        // for that, for its value is 2^94 and more times smaller than the unit, the unit comes down. A wave has one unit: F32 holds the sums of
        // weights of a head whose largest values count and of one whose smallest do if those are at most some 2^180 apart.
        float sum, largest;
        const auto weigh = [&] {
          const float base = m == -INFINITY ? 0.0f : m;
          sum = largest = 0.0f;
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            // Rounded as in the reference: where a score is past 2^30, what is left of it would be more than a weight can hold.
#pragma clang fp contract(off)
            const float sc = d[j] * factor;
            weight[j] = exp2_fast(sc - base);
          }
          if (!whole) {
#pragma unroll
            for (int j = 0; j < 8; ++j) weight[j] = j < valid ? weight[j] : 0.0f;
          }
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            sum += weight[j];
            const float w = weight[j] * ls[j];
            largest = fmaxf(largest, w);
            ratio_weight[j] = (_Float16)w;
          }
        };
        weigh();
        const bool raise = largest > 16384.0f || sum > 0x1p100f || m == -INFINITY;
        if (__any(raise)) {
          float top = -INFINITY, high = -INFINITY;
#pragma unroll
          for (int j = 0; j < 8; ++j) {
#pragma clang fp contract(off)
            const float sc = j < valid ? d[j] * factor : -INFINITY;
            top = fmaxf(top, sc);
            const int power = (int)(__float_as_uint(ls[j]) >> 23);
            high = fmaxf(high, sc + (float)(power == kNoScale ? kLeast : power - 127));
          }
          // Of the columns that need it: while the unit stays, a head's sums do not depend on the heads beside it.
          const bool own_raise = column_max(raise ? 1.0f : 0.0f) > 0.0f;
          // 2^6 for the largest weight exactly: where it is most of a softmax, as it often is, its rounding to F16 would be most of the error
          // (attention over 100 positions: off by 2.4e-4, with whole numbers 3.3e-4).
          const float largest_of_column = column_max(high), top_of_column = column_max(top);
          float from = (fabsf(largest_of_column) < 4096.0f ? largest_of_column : ceilf(largest_of_column)) - 6.0f;
          const float least = own_raise ? ceilf(top_of_column) - 100.0f : -INFINITY;
          if (__any(least > from && least > m)) {
            // The scales' unit comes down by what is missing, as far as the tile's largest allows.
            const int held = (int)(__float_as_uint(largest_scale[own]) >> 23);
            const int by = min(largest_of(least > from && least > m ? (int)(least - from) + 1 : 0), 254 - largest_of(held));
            move_unit(-by);
            from += (float)by;
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            if (held != kNoScale) largest_scale[own] = __uint_as_float((uint32_t)(held + by) << 23);
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            load8(largest_scale + 32 * s + 8 * quad, ls);
          }
          const float raised = own_raise ? fmaxf(m, fmaxf(from, least)) : m;
          // Twice the root: a sum of up to 2^127 may count beside 2^(m - raised) below F32's range.
          const float root = raised == m ? 1.0f : exp2_fast(0.5f * (m - raised)), rescale = root * root;
#pragma unroll
          for (int f = 0; f < 2 * G; ++f) o[f] *= rescale;
          l = l * root * root;
          m = raised;
          weigh();
        }
        l += sum;
      } else {
        // F32 tensors keep the scores' factor as a sum of two floats and round a score once, after the maximum is taken away.
        float sc[8], by_lo[8], most = -INFINITY;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          sc[j] = d[j] * factor;
          // Past 2^24 it is more than 1, and past 2^31 more than a weight can hold: scores are as good as F32's there.
          by_lo[j] = j >= valid || sc[j] == -INFINITY ? 0.0f : __builtin_amdgcn_fmed3f(fmaf(d[j], factor, -sc[j]) + d[j] * factor_lo, -1.0f, 1.0f);
          sc[j] = j < valid ? sc[j] : -INFINITY;
          most = fmaxf(most, sc[j]);
        }
        const float m_new = fmaxf(m, column_max(most));
        const float base = m_new == -INFINITY ? 0.0f : m_new;
        const float decay = exp2_fast(m - base);
        float sum = 0.0f, largest = 0.0f;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
#pragma clang fp contract(off)
          weight[j] = exp2_fast((sc[j] - base) + by_lo[j]);
          sum += weight[j];
          largest = fmaxf(largest, weight[j] * ls[j]);
        }
        l = l * decay + sum;
        m = m_new;
        r *= decay;
        largest = column_max(largest);
        if (__any(largest > 4096.0f * r)) {
          const float raised = fmaxf(r, largest), rescale = raised > r ? r / raised : 1.0f;
#pragma unroll
          for (int f = 0; f < 2 * G; ++f) o[f] *= rescale;
          r = raised;
        }
        const float over = r > 0x1p-125f ? __builtin_amdgcn_rcpf(r) : 0.0f;  // smaller weights are nothing
#pragma unroll
        for (int j = 0; j < 8; ++j) weight[j] *= over;
      }
#pragma unroll
      for (int w = 0; w < W; ++w) {
        // Two positions' codes are paired. E2M1: pairs[e] holds code e (of two) of both in each group's byte; INT4: pairs[k] both
        // positions' bytes of groups 2 k and 2 k + 1.
        uint32_t pairs[2][4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint32_t x = vw[2 * j][w], y = vw[2 * j + 1][w];
          if constexpr (F == kE2m1) {
            pairs[0][j] = (x & 0x0f0f0f0fu) | (y << 4 & 0xf0f0f0f0u);
            pairs[1][j] = (x >> 4 & 0x0f0f0f0fu) | (y & 0xf0f0f0f0u);
          } else {
            pairs[0][j] = __builtin_amdgcn_perm(y, x, 0x05040100u);
            pairs[1][j] = __builtin_amdgcn_perm(y, x, 0x07060302u);
          }
        }
#pragma unroll
        for (int gw = 0; gw < (G < 4 ? G : 4); ++gw) {
          const int g = 4 * w + gw;
          half8 pf[P];
          if constexpr (kRatios) {
            pf[0] = ratio_weight * ratios[g];
          } else {
            float vs[8];
            load8(reinterpret_cast<const float*>(value_scale) + g * N + 32 * s + 8 * quad, vs);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              float x = weight[j] * vs[j];
              // As a value of its own: rounded with the product in one step, the first part would differ
              // from the one that the second part is the rest of.
              asm("" : "+v"(x));
              pf[0][j] = (_Float16)x;
              pf[P - 1][j] = (_Float16)(x - (float)pf[0][j]);
            }
          }
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            half8 v;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              half2v x;
              if constexpr (F == kE2m1) {
                x = gw == 0   ? __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(pairs[e][j], 1.0f, 0)
                    : gw == 1 ? __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(pairs[e][j], 1.0f, 1)
                    : gw == 2 ? __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(pairs[e][j], 1.0f, 2)
                              : __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(pairs[e][j], 1.0f, 3);
              } else {
                const uint32_t two = gw & 1 ? pairs[gw >> 1][j] >> 8 : pairs[gw >> 1][j];
                x = e ? high_halves(two) : low_halves(two);
              }
              v[2 * j] = x[0];
              v[2 * j + 1] = x[1];
            }
#pragma unroll
            for (int p = P - 1; p >= 0; --p) o[2 * g + e] = mfma(v, pf[p], o[2 * g + e]);
          }
        }
      }
    }
  }

  // The four waves' states meet in LDS, each wave's in its own tile.
  l = column_sum(l);
  if constexpr (kRatios) {
    // References may lie far from their scores, by wave: the sum's exponent goes over to it, or 2^(m - another wave's) could be nothing
    // where the sum beside it is not.
    const int power = l > 0.0f && l < INFINITY && moves() ? (int)(__float_as_uint(l) >> 23) - 127 : 0;
    l = __builtin_amdgcn_ldexpf(l, -power);
    m += (float)power;
    r = unit == kNoUnit ? 0.0f : __builtin_amdgcn_ldexpf(1.0f, unit - 127 - power);
  }
  // Only scores of -inf (an infinite query's): a sum that is not 0 beside that maximum tells them from no positions.
  if (any && l == 0.0f) l = 1.0f;
  if (quad == 0) {
    states[wave][0][col] = m;
    states[wave][1][col] = l;
    states[wave][2][col] = r;
  }
  static_assert(Layout::kBytes >= 64 * D, "a wave's sums lie in its tile");
  // Components 2 k and 2 k + 1 of a group's two fragments: four elements that follow one another.
#pragma unroll
  for (int g = 0; g < G; ++g)
#pragma unroll
    for (int k = 0; k < 2; ++k)
      reinterpret_cast<floatx4*>(tile)[(2 * g + k) * 64 + lane] =
          floatx4{o[2 * g][2 * k], o[2 * g + 1][2 * k], o[2 * g][2 * k + 1], o[2 * g + 1][2 * k + 1]};
  __syncthreads();
  T* out = at<T>(a.out, row, kvh * a.group + g0, 0);
  if (a.cuts && low == 0 && threadIdx.x == 0) a.cuts[row * in_row + kvg] = int2{first, parts};
  for (int e = threadIdx.x; e < vectors * (D / 4); e += kThreads) {
    const int v = e / (D / 4), dim = e % (D / 4) * 4;
    const int from = ((dim / 32 * 2 + dim / 4 % 2) * 64 + dim % 32 / 8 * 16) + v;
    float top = -INFINITY, total = 0.0f, sums = 0.0f;
    floatx4 x[4];
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      x[w] = reinterpret_cast<const floatx4*>(smem + w * Layout::kBytes)[from];
      top = fmaxf(top, states[w][0][v]);
      sums += states[w][1][v];
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
    const bool undefined = total == 0.0f && sums != 0.0f;  // no softmax of scores that are all -inf
    if (parts == 1) {
      store4(out + v * a.out.head + dim, undefined ? floatx4{NAN, NAN, NAN, NAN} : y);
    } else {
      if (undefined) total = 1.0f;  // NaN in the join, unless another part has finite scores
      const uint64_t part = part_at(a, first, me - first, member, v);
      *reinterpret_cast<floatx4*>(a.part + part * D + dim) = y;
      if (dim == 0) *reinterpret_cast<float2*>(a.stats + 2 * part) = float2{top, total};
    }
  }
  }
}

template <typename T, int F>
void kv4_read(hipStream_t stream, int head_dim, const ReadArgs& a) {
  const uint64_t units = (uint64_t)a.rows * a.pages.kv_heads * (head_dim * sizeof(T) / 16);
  const unsigned blocks = (unsigned)((units + kThreads - 1) / kThreads);
  if (head_dim == 64) kv4_read_kernel<T, F, 64><<<blocks, kThreads, 0, stream>>>(a);
  if (head_dim == 128) kv4_read_kernel<T, F, 128><<<blocks, kThreads, 0, stream>>>(a);
  if (head_dim == 256) kv4_read_kernel<T, F, 256><<<blocks, kThreads, 0, stream>>>(a);
}

template <typename T, int F, int D>
void attend4(hipStream_t stream, const AttendArgs& a) {
  constexpr int kLds = Tile4<T, F, D>::kBlock;
  static std::atomic<uint64_t> asked{0};
  ask_for_lds(reinterpret_cast<const void*>(&kv4_attention_kernel<T, F, D>), kLds, asked);
  const int round = 8 * a.cluster;
  kv4_attention_kernel<T, F, D><<<(a.blocks + round - 1) / round * round, kThreads, kLds, stream>>>(a);
}

template <typename T, int F>
void attend4_dim(hipStream_t stream, int head_dim, const AttendArgs& a) {
  if (head_dim == 64) attend4<T, F, 64>(stream, a);
  if (head_dim == 128) attend4<T, F, 128>(stream, a);
  if (head_dim == 256) attend4<T, F, 256>(stream, a);
}

template <typename F>
void by_dtype(uint32_t dtype, F&& run) {
  if (dtype == HLLM_DTYPE_F16) return run(_Float16{});
  if (dtype == HLLM_DTYPE_BF16) return run(bhalf{});
  run(0.0f);
}

}  // namespace

void launch_kv4_read(hipStream_t stream, uint32_t dtype, int format, int head_dim, const ReadArgs& a) {
  by_dtype(dtype, [&](auto zero) {
    using T = decltype(zero);
    if (format == kE2m1)
      kv4_read<T, kE2m1>(stream, head_dim, a);
    else
      kv4_read<T, kInt4>(stream, head_dim, a);
  });
}

void launch_kv4_attention(hipStream_t stream, uint32_t dtype, int format, int head_dim, const AttendArgs& a) {
  by_dtype(dtype, [&](auto zero) {
    using T = decltype(zero);
    if (format == kE2m1)
      attend4_dim<T, kE2m1>(stream, head_dim, a);
    else
      attend4_dim<T, kInt4>(stream, head_dim, a);
  });
}

}  // namespace hllm_rocm
