// Operators on a caller's device memory: rotary positions, the 8-bit paged KV cache (written and
// read back), and one new token's attention over it. The C entry points are at the end.
#include "operators.hpp"

#include <algorithm>
#include <cmath>

#include "abi.hpp"

namespace hllm_rocm {
namespace {

constexpr int kThreads = 256;
constexpr float kLog2e = 1.4426950408889634f;

typedef __bf16 bhalf;
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
// product is its low 64 bits, of which the upper 32 are kept (2^-32 turn is 1.5e-9). Reduced to
// the nearest quarter turn, |x| <= pi / 4, where the Taylor series to x^9 and x^8 are off by at
// most 2e-9 and 3e-8.
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
// every pair is read before it is written and a tensor can be rotated in place.
//
// F >= 0: q_out is written as above, k is rotated and k and v are quantised: a head's lanes
// share its largest value by shuffles.
template <typename T, int F, bool kExchange>
__global__ void __launch_bounds__(kThreads) rotate_kernel(RotateArgs a) {
  __shared__ float2 cs[128];
  __shared__ float xs[kExchange ? kThreads * 17 : 1];
  const int row = blockIdx.x, t = threadIdx.x;
  int slot = 0;
  if constexpr (F >= 0) {
    slot = uniform_load(a.slots + row);
    if (slot < 0 || (slot >> a.pages.page_shift) >= a.pages.pages) return;
  }
  const int R = a.rotary, half = R / 2;
  const int in_block = t / a.lanes, u = t - in_block * a.lanes;
  const int head = blockIdx.y * a.heads_per_block + in_block;
  const bool active = in_block < a.heads_per_block && head < a.q_heads + a.k_heads + a.v_heads;
  const bool is_q = head < a.q_heads, is_v = head >= a.q_heads + a.k_heads;
  const int h = is_q ? head : is_v ? head - a.q_heads - a.k_heads : head - a.q_heads;
  const bool paired = !kExchange && !a.interleaved && !is_v && 16 * u < R;
  const int d0 = paired ? 8 * u : 16 * u, d1 = paired ? half + 8 * u : 16 * u + 8;
  float x[16];
  if (active) {
    const Strided& in = is_q ? a.q : is_v ? a.v : a.k;
    load8(at<const T>(in, row, h, d0), x);
    load8(at<const T>(in, row, h, d1), x + 8);
  }
  if (t < half) {
    const float2 v = turn(uniform_load(a.positions + row), a.turns[t]);
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
        if (16 * u + 2 * i >= R) continue;
        const float2 v = cs[8 * u + i];
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

// A thread reads sixteen codes of a key and of the value beside it and writes them: nothing
// but memory traffic.
template <typename T, int F, int D>
__global__ void __launch_bounds__(kThreads) kv_read_kernel(ReadArgs a) {
  constexpr int L = D / 16;
  const Pages& c = a.pages;
  const uint32_t per_row = (uint32_t)c.kv_heads * L;
  const uint64_t unit = (uint64_t)blockIdx.x * kThreads + threadIdx.x;
  const uint64_t row = unit / per_row;
  if (row >= (uint64_t)a.rows) return;
  const int in_row = (int)(unit - row * per_row), h = in_row / L, d = in_row % L * 16;
  const int slot = a.slots[row];
  if (slot < 0 || (slot >> c.page_shift) >= c.pages) return;
  const int page = slot >> c.page_shift, offset = slot & ((1 << c.page_shift) - 1);
  const uint64_t from = (uint64_t)page * c.page_stride + (uint64_t)offset * c.token_stride + (uint64_t)h * c.head_stride + d;
  const uint64_t scale_at = (((uint64_t)page * c.kv_heads + h) << c.page_shift) + offset;
  const uint4v codes[2] = {*reinterpret_cast<const uint4v*>(c.keys + from), *reinterpret_cast<const uint4v*>(c.values + from)};
  const float scale[2] = {c.key_scales[scale_at], c.value_scales[scale_at]};
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    float x[16];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const floatx4 v = decode4<F>(codes[which][j]);
#pragma unroll
      for (int i = 0; i < 4; ++i) x[4 * j + i] = v[i] * scale[which];
    }
    T* to = at<T>(which ? a.v : a.k, (int)row, h, d);
    store8(to, x);
    store8(to + 8, x + 8);
  }
}

// ---------------------------------------------------------------- attention

__device__ inline floatx4 mfma(half8 a, half8 b, floatx4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}
__device__ inline float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }
// The largest of a value over the four lanes of a column (lanes 16 apart).
__device__ inline float column_max(float v) {
  v = fmaxf(v, __shfl_xor(v, 16, 64));
  return fmaxf(v, __shfl_xor(v, 32, 64));
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

template <typename T, int F, int D>
__global__ void __launch_bounds__(kThreads) kv_attention_kernel(AttendArgs a) {
  constexpr int KK = D / 32;   // 32-wide chunks of the score contraction
  constexpr int DF = D / 16;   // 16-row fragments of the output; a lane's value bytes of a position
  constexpr int VW = DF / 4;   // ... in words
  constexpr int P = sizeof(T) == 4 ? 2 : 1;  // F16 parts of a query element and of a weight
  __shared__ int32_t held[kAttendMostKeys / 8 + 1];
  __shared__ float merge[4 * 4 * DF * 64];
  __shared__ float states[4][3][16];

  const Pages& c = a.pages;
  const int KVH = c.kv_heads, shift = c.page_shift;
  const int pairs = a.rows * KVH * a.head_groups;
  const int split = blockIdx.x / pairs, pair = blockIdx.x - split * pairs;
  const int row = pair / (KVH * a.head_groups), kvg = pair - row * KVH * a.head_groups;
  const int kvh = kvg / a.head_groups, g0 = (kvg - kvh * a.head_groups) * 16;
  const int stated = uniform_load(a.lengths + row);
  if (stated < 0) return;
  const int length = min(stated, a.limit);
  const int per = attend_part(length, a.splits, a.unit);
  const int begin = split * per;
  if (begin >= length && split > 0) return;
  const int end = min(length, begin + per);
  const int parts = (length + per - 1) / per;

  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int quad = lane >> 4, col = lane & 15;
  const int vectors = min(16, a.group - g0);

  // The part's page numbers, -1 for those that name no page.
  const int first_page = begin >> shift, held_pages = ((end - 1) >> shift) - first_page + 1;
  for (int i = threadIdx.x; i < held_pages; i += kThreads) {
    const int id = a.table[(uint64_t)row * a.table_stride + first_page + i];
    held[i] = id >= 0 && id < c.pages ? id : -1;
  }

  // Q^T as the B operand: chunk kk = 2 hh + s holds elements 64 hh + 16 quad + 8 s + j, the order
  // of a key's sixteen bytes. Each vector is divided by the power of two of its
  // largest element, which puts F32 and BF16 ranges into F16's and goes back into its scores.
  half8 qf[P][KK];
  float factor;
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
    // 2^e <= largest < 2^(e+1), for e from -126 to 126; other vectors (zero, not finite) as they are.
    const uint32_t exponent = most >> 23;
    const bool usual = exponent >= 1 && exponent <= 253;
    const float down = usual ? __uint_as_float((254u - exponent) << 23) : 1.0f;
    factor = a.scale * kLog2e * (usual ? __uint_as_float(exponent << 23) : 1.0f);
#pragma unroll
    for (int kk = 0; kk < KK; ++kk)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float y = x[kk][j] * down;
        qf[0][kk][j] = (_Float16)y;
        if constexpr (P == 2) qf[1][kk][j] = (_Float16)(y - (float)qf[0][kk][j]);
      }
  }
  __syncthreads();

  // The weights of a position are 2^(score - m) times its value scale; they enter the products
  // divided by their running maximum r, and so do the sums o.
  floatx4 o[DF];
#pragma unroll
  for (int f = 0; f < DF; ++f) o[f] = floatx4{0.f, 0.f, 0.f, 0.f};
  float m = -INFINITY, l = 0.0f, r = 0.0f;

  const uint64_t head_at = (uint64_t)kvh * c.head_stride;
  const uint8_t* keys = c.keys + head_at + 16 * quad;
  const uint8_t* values = c.values + head_at + DF * col;
  const int mask = (1 << shift) - 1;
  const uint64_t token = c.token_stride;
  for (int t = begin + 32 * wave; t < end; t += 128) {
    // Score fragment h's row 4 q + i is position 8 q + 4 h + i: a lane's scores are the eight
    // positions 8 quad .. + 7, which are also its slots of the value products.
    const int key_at = t + 8 * (col >> 2), own_at = t + 8 * quad;
    const int key_page = held[min((key_at >> shift) - first_page, held_pages - 1)];
    const int own_page = held[min((own_at >> shift) - first_page, held_pages - 1)];
    const uint8_t* kp = keys + (uint64_t)max(key_page, 0) * c.page_stride + (uint64_t)((key_at & mask) + (col & 3)) * token;
    const uint8_t* vp = values + (uint64_t)max(own_page, 0) * c.page_stride + (uint64_t)(own_at & mask) * token;
    const uint64_t scale_at = (((uint64_t)max(own_page, 0) * KVH + kvh) << shift) + (own_at & mask);
    uint4v kw[2][D / 64];
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int hh = 0; hh < D / 64; ++hh) kw[h][hh] = *reinterpret_cast<const uint4v*>(kp + 4 * h * token + 64 * hh);
    uint32_t vw[8][VW];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if constexpr (VW == 1) vw[j][0] = *reinterpret_cast<const uint32_t*>(vp + j * token);
      if constexpr (VW == 2) {
        const uint2v w = *reinterpret_cast<const uint2v*>(vp + j * token);
        vw[j][0] = w[0];
        vw[j][1] = w[1];
      }
      if constexpr (VW == 4) {
        const uint4v w = *reinterpret_cast<const uint4v*>(vp + j * token);
#pragma unroll
        for (int i = 0; i < 4; ++i) vw[j][i] = w[i];
      }
    }
    float ks[8], vs[8];
    load8(c.key_scales + scale_at, ks);
    load8(c.value_scales + scale_at, vs);

    floatx4 s0 = {0.f, 0.f, 0.f, 0.f}, s1 = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int kk = 0; kk < KK; ++kk) {
      half8 k[2];
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int w = 0; w < 2; ++w) {
          half2v lo, hi;
          halves4<F>(kw[h][kk >> 1][2 * (kk & 1) + w], lo, hi);
          k[h][4 * w] = lo[0];
          k[h][4 * w + 1] = lo[1];
          k[h][4 * w + 2] = hi[0];
          k[h][4 * w + 3] = hi[1];
        }
#pragma unroll
      for (int p = 0; p < P; ++p) {
        s0 = mfma(k[0], qf[p][kk], s0);
        s1 = mfma(k[1], qf[p][kk], s1);
      }
    }
    float sc[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      sc[i] = s0[i] * (ks[i] * factor);
      sc[4 + i] = s1[i] * (ks[4 + i] * factor);
    }
    // Positions past the part and in pages that are not there: whatever their memory holds.
    const int valid = own_page < 0 ? 0 : end - own_at;
    if (__any(valid < 8)) {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (i >= valid) {
          sc[i] = -INFINITY;
          vs[i] = 0.0f;
#pragma unroll
          for (int w = 0; w < VW; ++w) vw[i][w] = 0;
        }
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
      const float p = exp2_fast(sc[i] - base);
      sum += p;
      weight[i] = p * vs[i];
      largest = fmaxf(largest, weight[i]);
    }
    l = l * decay + sum;
    m = m_new;
    const float r_old = r * decay;
    r = fmaxf(r_old, column_max(largest));
    const float over = r > 0x1p-120f ? 1.0f / r : 0.0f;  // smaller sums are nothing
    const float rescale = r_old * over;
    half8 pf[P];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float w = weight[i] * over;
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
      for (int i = 0; i < 4; ++i) {
        floatx4 acc = o[4 * w + i] * rescale;
#pragma unroll
        for (int p = 0; p < P; ++p) acc = mfma(v[i], pf[p], acc);
        o[4 * w + i] = acc;
      }
    }
  }

  // The four waves' states meet in LDS; wave i then sums and writes the elements of the
  // accumulators' component i.
  l = column_sum(l);
  if (quad == 0) {
    states[wave][0][col] = m;
    states[wave][1][col] = l;
    states[wave][2][col] = r;
  }
#pragma unroll
  for (int f = 0; f < DF; ++f)
#pragma unroll
    for (int i = 0; i < 4; ++i) merge[((wave * 4 + i) * DF + f) * 64 + lane] = o[f][i];
  __syncthreads();
  float top = -INFINITY;
#pragma unroll
  for (int w = 0; w < 4; ++w) top = fmaxf(top, states[w][0][col]);
  const float base = top == -INFINITY ? 0.0f : top;
  float total = 0.0f, share[4];
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    const float decay = exp2_fast(states[w][0][col] - base);
    total += states[w][1][col] * decay;
    share[w] = states[w][2][col] * decay;
  }
  if (col >= vectors) return;
  const float over = total == 0.0f ? 0.0f : 1.0f / total;
  float y[DF];
#pragma unroll
  for (int f = 0; f < DF; ++f) {
    float s = 0.0f;
#pragma unroll
    for (int w = 0; w < 4; ++w) s += merge[((w * 4 + wave) * DF + f) * 64 + lane] * share[w];
    y[f] = s * over;
  }
  const int head = kvh * a.group + g0 + col, d = 4 * DF * quad + DF * wave;
  if (parts > 1) {
    const uint64_t part = ((uint64_t)row * a.q_heads + head) * a.splits + split;
    float* to = a.part + part * D + d;
#pragma unroll
    for (int f = 0; f < DF; f += 4) *reinterpret_cast<floatx4*>(to + f) = floatx4{y[f], y[f + 1], y[f + 2], y[f + 3]};
    if (quad == 0 && wave == 0) {
      a.stats[2 * part] = top;
      a.stats[2 * part + 1] = total;
    }
  } else {
    T* to = at<T>(a.out, row, head, d);
    if constexpr (DF >= 8) {
#pragma unroll
      for (int f = 0; f < DF; f += 8) store8(to + f, y + f);
    } else {
#pragma unroll
      for (int f = 0; f < DF; ++f) to[f] = (T)y[f];
    }
  }
}

// Joins a row's parts, one workgroup for a query head: each part's output weighted with its
// share of the softmax sum.
template <typename T, int D>
__global__ void __launch_bounds__(kThreads) kv_join_kernel(AttendArgs a) {
  constexpr int L = D / 4, kSlots = kThreads / L;  // lanes of a part's vector; parts at a time
  __shared__ float sums[kSlots][D];
  __shared__ float totals[kSlots];
  const int row = blockIdx.x / a.q_heads, head = blockIdx.x - row * a.q_heads;
  const int length = min(uniform_load(a.lengths + row), a.limit);
  if (length <= 0) return;
  const int per = attend_part(length, a.splits, a.unit), parts = (length + per - 1) / per;
  if (parts <= 1) return;
  const uint64_t first = (uint64_t)blockIdx.x * a.splits;
  const float* stats = a.stats + 2 * first;
  float top = -INFINITY;
  for (int s = threadIdx.x & 63; s < parts; s += 64) top = fmaxf(top, stats[2 * s]);
  for (int o = 32; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o, 64));
  const float base = top == -INFINITY ? 0.0f : top;
  const int slot = threadIdx.x / L, d = threadIdx.x % L * 4;
  floatx4 sum = {0.f, 0.f, 0.f, 0.f};
  float total = 0.0f;
#pragma unroll 4
  for (int s = slot; s < parts; s += kSlots) {
    const float share = exp2_fast(stats[2 * s] - base) * stats[2 * s + 1];
    total += share;
    sum += *reinterpret_cast<const floatx4*>(a.part + (first + s) * D + d) * share;
  }
  *reinterpret_cast<floatx4*>(&sums[slot][d]) = sum;
  if (d == 0) totals[slot] = total;
  __syncthreads();
  if (threadIdx.x >= D) return;
  float y = 0.0f, all = 0.0f;
#pragma unroll
  for (int s = 0; s < kSlots; ++s) {
    y += sums[s][threadIdx.x];
    all += totals[s];
  }
  *at<T>(a.out, row, head, threadIdx.x) = (T)(all == 0.0f ? 0.0f : y / all);
}

template <typename T, int F>
void rotate(hipStream_t stream, int rows, const RotateArgs& a) {
  const int heads = a.q_heads + a.k_heads + a.v_heads;
  const int threads = std::min(kThreads, (heads * a.lanes + 63) / 64 * 64);
  RotateArgs b = a;
  b.heads_per_block = threads / a.lanes;
  const dim3 grid(rows, (heads + b.heads_per_block - 1) / b.heads_per_block);
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
  const uint64_t units = (uint64_t)a.rows * a.pages.kv_heads * (head_dim / 16);
  const unsigned blocks = (unsigned)((units + kThreads - 1) / kThreads);
  if (head_dim == 64) kv_read_kernel<T, F, 64><<<blocks, kThreads, 0, stream>>>(a);
  if (head_dim == 128) kv_read_kernel<T, F, 128><<<blocks, kThreads, 0, stream>>>(a);
  if (head_dim == 256) kv_read_kernel<T, F, 256><<<blocks, kThreads, 0, stream>>>(a);
}

template <typename T, int F, int D>
void attend(hipStream_t stream, const AttendArgs& a) {
  const unsigned blocks = (unsigned)((uint64_t)a.rows * a.pages.kv_heads * a.head_groups * a.splits);
  kv_attention_kernel<T, F, D><<<blocks, kThreads, 0, stream>>>(a);
  if (a.splits > 1) kv_join_kernel<T, D><<<(unsigned)(a.rows * a.q_heads), kThreads, 0, stream>>>(a);
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

// Rows of one call: grids stay below 2^32 threads.
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

void check_rows(uint64_t rows) {
  if (rows > kMostRows) refuse("at most 1048576 rows a call");
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
  if (p->page_stride > (1ull << 40) || p->token_stride > (1ull << 40) || p->head_stride > (1ull << 40))
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
          p->pages > 1 ? p->page_stride : 0, p->token_stride, head, (int32_t)p->pages, shift, (int32_t)p->kv_heads};
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
  }
  for (uint32_t i = 0; i < n / 2; ++i) {
    long double f = std::pow((long double)c.theta, -2.0L * i / n);
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
    take_rope(rope, positions, a);
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
    if (rope) take_rope(rope, positions, a);
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
    if (rows * pages->kv_heads * (pages->head_dimension / 16) > kMostBlocks * kThreads) refuse("too many rows for these heads");
    OnDevice on(device);
    launch_kv_read(static_cast<hipStream_t>(stream), k_out->dtype, (int)pages->format, (int)pages->head_dimension, a);
    HIP_CHECK(hipGetLastError());
  });
}

}  // extern "C"

namespace {

// The split of a call and the floats of its workspace.
struct AttendPlan {
  uint64_t head_groups = 1;
  AttendSplit split{1, 1};
  uint64_t parts = 0;  // [rows][query_heads][splits], 0 when rows are not split
  uint64_t bytes = 0;
};

AttendPlan plan_attention(const hllm_rocm_kv_pages& pages, uint64_t rows, uint64_t query_heads, uint64_t limit) {
  if (query_heads < 1 || query_heads > 1024 || query_heads % pages.kv_heads)
    refuse("query heads are a multiple of the cache's heads, at most 1024");
  AttendPlan p;
  if (rows == 0) return p;
  p.head_groups = (query_heads / pages.kv_heads + 15) / 16;
  const uint64_t pairs = rows * pages.kv_heads * p.head_groups;
  p.split = attend_split(pairs, limit);
  if (pairs * p.split.splits > kMostBlocks || rows * query_heads > kMostBlocks) refuse("too many rows for these heads and lengths");
  if (p.split.splits > 1) {
    p.parts = rows * query_heads * p.split.splits;
    p.bytes = p.parts * (pages.head_dimension + 2) * sizeof(float);
  }
  return p;
}

uint64_t clamp_length(uint64_t max_length) { return std::min<uint64_t>(max_length, 0x7fffffffull); }

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
    if (!std::isfinite(args->scale)) refuse("scale is not finite");
    if (!args->lengths) refuse("lengths is null");
    if (args->table_width > 0x7fffffffull / pages->page_tokens) refuse("a page table's row holds at most 2^31 - 1 positions");
    const uint64_t limit = std::min(clamp_length(args->max_length), args->table_width * pages->page_tokens);
    if (limit > 0 && !args->page_table) refuse("page_table is null");
    if (args->table_stride > (1ull << 40)) refuse("table_stride is too large");
    const AttendPlan plan = plan_attention(*pages, rows, args->q.heads, limit);
    if (plan.bytes > 0 && (!args->workspace || args->workspace_bytes < plan.bytes || (uintptr_t)args->workspace % 16))
      refuse("the workspace is null, not 16-byte aligned or below " + std::to_string(plan.bytes) + " bytes");
    a.table = args->page_table;
    a.table_stride = args->table_stride;
    a.lengths = args->lengths;
    a.rows = (int32_t)rows;
    a.q_heads = (int32_t)args->q.heads;
    a.group = a.q_heads / a.pages.kv_heads;
    a.head_groups = (int32_t)plan.head_groups;
    a.limit = (int32_t)limit;
    a.splits = plan.split.splits;
    a.unit = plan.split.unit;
    a.scale = args->scale;
    a.part = static_cast<float*>(args->workspace);
    a.stats = a.part + plan.parts * D;
    OnDevice on(device);
    launch_kv_attention(static_cast<hipStream_t>(stream), args->q.dtype, (int)pages->format, (int)D, a);
    HIP_CHECK(hipGetLastError());
  });
}

}  // extern "C"
