// What the kernels of caches of 8 and 4 bits share (kv_8bit.cu, kv_4bit.cu, tree_attn.cu): where a head's numbers lie, and the views' checks.
#pragma once
#include "common.cuh"

namespace {

constexpr int GROUP4 = 32;                                         // channels that share a scale in a cache of 4 bits

// A cache as the kernels take it: strides in bytes for data, in numbers for scales
struct Cache8 {
  uint8_t* data;
  float* scale;                                                    // (of 4 bits: bf16, by scale4_at)
  long long slot, pos, head, scale_slot, scale_head;
  int slots, capacity, dim;

  __device__ __forceinline__ bool holds(int s, int p) const { return (unsigned)s < (unsigned)slots && (unsigned)p < (unsigned)capacity; }
  __device__ __forceinline__ uint8_t* at(int s, int p, int h) const { return data + s * slot + p * pos + h * head; }
  __device__ __forceinline__ float* scale_at(int s, int h) const { return scale + s * scale_slot + h * scale_head; }
  // of 4 bits: dim / GROUP4 scales for each position
  __device__ __forceinline__ bf16* scale4_at(int s, int h) const { return reinterpret_cast<bf16*>(scale) + s * scale_slot + h * scale_head; }
};

// Of 4 bits: the number of channel c of a head is in byte byte4() of its dim / 2, as code + 8 in the lower four bits (c even) or the upper ones: four neighbouring channels of a group are two bytes, and
// those of all groups at the same place in them lie side by side, so that a lane that takes neighbouring bytes has channels of every group
__host__ __device__ __forceinline__ int byte4(int c, int dim) { return ((c % GROUP4 / 4) * (dim / GROUP4) + c / GROUP4) * 2 + c % 4 / 2; }

inline Cache8 cache8(const LiaCacheView* v) {
  const long long b = v->type == LIA_CACHE_BF16 ? 2 : 1;
  return {reinterpret_cast<uint8_t*>(v->data), reinterpret_cast<float*>(v->scale), v->slot_stride * b, v->pos_stride * b, v->head_stride * b, v->scale_slot_stride, v->scale_head_stride, v->slots, v->capacity, v->dim};
}

// NULL, or what is wrong with a view whose addresses are to be multiples of `align` bytes
inline const char* cache8_wrong(const LiaCacheView* v, int align) {
  if (!v || !v->data) return "null cache";
  if (v->type < LIA_CACHE_BF16 || v->type > LIA_CACHE_INT4) return "unknown type of cache";
  if ((v->type != LIA_CACHE_BF16) != (v->scale != nullptr)) return "scales go with caches of 8 and 4 bits, and with no other";
  if (v->slots <= 0 || v->capacity <= 0 || v->dim <= 0) return "an empty cache";
  if (v->type == LIA_CACHE_INT4) {
    if (v->dim % GROUP4) return "heads of 4 bits have to be multiples of 32 channels";
    const int vec = v->dim / GROUP4 % 4 == 0 ? 4 : v->dim / GROUP4 % 2 == 0 ? 2 : 1;              // a position's scales are read so many at once
    if (reinterpret_cast<uintptr_t>(v->scale) % (2 * vec) || v->scale_slot_stride % vec || v->scale_head_stride % vec) return "scales of 4-bit heads that are not whole vectors apart";
  }
  const long long b = v->type == LIA_CACHE_BF16 ? 2 : 1;
  if (reinterpret_cast<uintptr_t>(v->data) % align || v->slot_stride * b % align || v->pos_stride * b % align || v->head_stride * b % align) return "a cache whose heads are not whole vectors apart";
  return nullptr;
}

}  // namespace
