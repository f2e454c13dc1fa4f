// What the kernels of 8-bit caches share (kv_8bit.cu, tree_attn.cu): where a head's numbers lie, and the views' checks.
#pragma once
#include "common.cuh"

namespace {

// A cache as the kernels take it: strides in bytes for data, in numbers for scales
struct Cache8 {
  uint8_t* data;
  float* scale;
  long long slot, pos, head, scale_slot, scale_head;
  int slots, capacity, dim;

  __device__ __forceinline__ bool holds(int s, int p) const { return (unsigned)s < (unsigned)slots && (unsigned)p < (unsigned)capacity; }
  __device__ __forceinline__ uint8_t* at(int s, int p, int h) const { return data + s * slot + p * pos + h * head; }
  __device__ __forceinline__ float* scale_at(int s, int h) const { return scale + s * scale_slot + h * scale_head; }
};

inline Cache8 cache8(const LiaCacheView* v) {
  const long long b = v->type == LIA_CACHE_BF16 ? 2 : 1;
  return {reinterpret_cast<uint8_t*>(v->data), v->scale, v->slot_stride * b, v->pos_stride * b, v->head_stride * b, v->scale_slot_stride, v->scale_head_stride, v->slots, v->capacity, v->dim};
}

// NULL, or what is wrong with a view whose addresses are to be multiples of `align` bytes
inline const char* cache8_wrong(const LiaCacheView* v, int align) {
  if (!v || !v->data) return "null cache";
  if (v->type < LIA_CACHE_BF16 || v->type > LIA_CACHE_E4M3) return "unknown type of cache";
  if ((v->type != LIA_CACHE_BF16) != (v->scale != nullptr)) return "scales go with 8-bit caches, and with no other";
  if (v->slots <= 0 || v->capacity <= 0 || v->dim <= 0) return "an empty cache";
  const long long b = v->type == LIA_CACHE_BF16 ? 2 : 1;
  if (reinterpret_cast<uintptr_t>(v->data) % align || v->slot_stride * b % align || v->pos_stride * b % align || v->head_stride * b % align) return "a cache whose heads are not whole vectors apart";
  return nullptr;
}

}  // namespace
