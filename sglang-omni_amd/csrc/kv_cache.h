// Shared pieces of the kernels around the paged key-value cache: where a slot's row lies, and the rows
// of each type it holds.
#pragma once

#include "block_fp8.h"

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));

// Workgroups of 256 threads that a launch can have: a grid's threads count in 32 bits.
constexpr int64_t kMostWorkgroups = 0xffffff;

// A cache as the kernels take it: rows [pages][kv_heads][page_size][dim], strides in elements (all
// below 2^31 rows, so slots are 32-bit).
struct CacheView {
  uint8_t* keys;
  uint8_t* values;
  float* key_scale;
  float* value_scale;
  int64_t page, head, token;                    // strides of the rows
  int64_t scale_page, scale_head, scale_token;  // strides of the scales
  int pages, page_size;
};

// false where the arguments cannot be a cache: a null row pointer, a type that is not held, sizes out
// of range, rows off their alignment.
inline bool cache_view(const omni_kv_cache& c, int64_t row_alignment, CacheView* v) {
  const int size = c.dtype == OMNI_DTYPE_FP8_E4M3 ? 1 : 2;
  if (c.dtype != OMNI_DTYPE_BF16 && c.dtype != OMNI_DTYPE_F16 && c.dtype != OMNI_DTYPE_FP8_E4M3)
    return false;
  if (!c.keys || !c.values || c.pages < 1 || c.page_size < 1 || c.pages > 0x7fffffffLL ||
      c.page_size > 0x7fffffffLL || c.pages * c.page_size > 0x7fffffffLL)
    return false;
  if (!aligned_to(c.keys, (int)row_alignment) || !aligned_to(c.values, (int)row_alignment) ||
      c.stride_page * size % row_alignment || c.stride_head * size % row_alignment ||
      c.stride_token * size % row_alignment)
    return false;
  if (c.dtype == OMNI_DTYPE_FP8_E4M3 &&
      (!c.key_scale || !c.value_scale || !aligned_to(c.key_scale, 4) || !aligned_to(c.value_scale, 4)))
    return false;
  v->keys = static_cast<uint8_t*>(c.keys);
  v->values = static_cast<uint8_t*>(c.values);
  v->key_scale = c.key_scale;
  v->value_scale = c.value_scale;
  v->page = c.stride_page;
  v->head = c.stride_head;
  v->token = c.stride_token;
  v->scale_page = c.scale_stride_page;
  v->scale_head = c.scale_stride_head;
  v->scale_token = c.scale_stride_token;
  v->pages = (int)c.pages;
  v->page_size = (int)c.page_size;
  return true;
}
