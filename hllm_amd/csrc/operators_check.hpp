// Checks of the operators' arguments that several entry points make.
#pragma once

#include <algorithm>
#include <type_traits>

#include "abi.hpp"
#include "operators.hpp"

namespace hllm_rocm {
namespace {

// Rows of one call, and workgroups of kThreads threads of one launch: below 2^32 threads over all of a grid's dimensions.
constexpr uint64_t kMostRows = 1u << 20;
constexpr uint64_t kMostBlocks = (1u << 24) - 1;

[[noreturn]] inline void refuse(const std::string& message) { fail(HLLM_INVALID_REQUEST, message); }

inline size_t element_size(uint32_t dtype) { return dtype == HLLM_DTYPE_F32 ? 4 : 2; }

// Whether vectors of `width` at strides a (of na) and b (of nb) are apart, one inside the other.
inline bool apart(uint64_t width, uint64_t na, uint64_t a, uint64_t nb, uint64_t b) {
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

inline Strided tensor(const hllm_rocm_tensor* t, const char* name, uint64_t rows, uint64_t width, bool output) {
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
inline void check_in_place(const hllm_rocm_tensor* in, const hllm_rocm_tensor* out, uint64_t rows) {
  if (in->data != out->data) return;
  if ((rows > 1 && in->row_stride != out->row_stride) || (in->heads > 1 && in->head_stride != out->head_stride))
    refuse("an output in its input's memory must have its strides");
}

// Two outputs, or an output and another tensor's input, that start at one address.
inline void check_apart(const void* a, const char* name_a, const void* b, const char* name_b) {
  if (a == b) refuse(std::string(name_a) + " and " + name_b + " are one memory");
}

inline void check_rows(uint64_t rows) {
  if (rows > kMostRows) refuse("at most 1048576 rows a call");
}

// Positions of one row: sums of a length and a tile's stay below 2^31.
constexpr uint64_t kMostPositions = 1u << 30;

// A cache of either kind as the entry points take it: T is hllm_rocm_kv_pages or hllm_rocm_kv4_pages.
template <typename T>
Cache cache_of(const T* p) {
  constexpr bool kFour = std::is_same_v<T, hllm_rocm_kv4_pages>;
  if (!p) refuse("pages is null");
  if (p->format > 1) refuse("unknown cache format");
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
  const uint64_t width = kFour ? p->head_dimension / 2 : p->head_dimension;  // bytes of a vector
  const uint64_t head = p->kv_heads > 1 ? p->head_stride : 0;
  const uint64_t extent = (p->page_tokens - 1) * p->token_stride + (p->kv_heads - 1) * head + width;
  if (!apart(width, p->page_tokens, p->token_stride, p->kv_heads, head) ||
      (p->pages > 1 && p->page_stride < extent))
    refuse("a cache's vectors overlap");
  int shift = 0;
  while ((1u << shift) < p->page_tokens) ++shift;
  const Pages pages = {static_cast<uint8_t*>(p->keys), static_cast<uint8_t*>(p->values), p->key_scales, p->value_scales,
                       p->pages > 1 ? (uint32_t)p->page_stride : 0u, (uint32_t)p->token_stride, head, (int32_t)p->pages, shift,
                       (int32_t)p->kv_heads};
  return {pages, (int)p->format + (kFour ? kE2m1 : 0), (int)p->head_dimension, p->page_tokens};
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

inline void check_device(int32_t device) {
  if (device < 0) refuse("device is negative");
}

}  // namespace
}  // namespace hllm_rocm
