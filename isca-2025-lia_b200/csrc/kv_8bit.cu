// Keys and values in 8 bits: quantised as they are written into a cache, and read back.
//
//   int8   a = max |x| over a head of one token, scale = a / 127, code = rint(127 x / a): an even grid, for heads whose numbers are alike
//   e4m3   scale = 2^e, the least with a / 2^e <= 448, code = x / 2^e rounded to 4 significant bits.  A float keeps its 4 bits at any of 15 powers of two, so a power of two
//          loses nothing against a / 448 down to a / 28672, and makes scaling and reading back exact.
// One scale for each head of each token: a token that comes later changes nothing that is there, and attention multiplies scores and weights by scales instead of channels by them.
//
// Both kernels move each number once and compute about ten operations on it, so memory bounds them.  A group of 8 to 32 neighbouring lanes has a head of a token, eight channels a
// lane: its largest magnitude takes three to five shuffles, and no shared memory.
#include <cuda_fp8.h>

#include "cache8.cuh"

namespace {

constexpr int THREADS = 256;
constexpr float LEAST = 7.888609052210118e-31f;                    // 2^-100: keeps scales and their inverses normal numbers

template <typename T> __device__ __forceinline__ void load8(const T* p, bool vec, float* f) {
  if constexpr (sizeof(T) == 2) {
    if (vec) {
      unpack8(ldg_act(p), f);
      return;
    }
  } else if (vec) {
    const uint4 u = ldg_act(p), w = ldg_act(p + 4);
    f[0] = __uint_as_float(u.x); f[1] = __uint_as_float(u.y); f[2] = __uint_as_float(u.z); f[3] = __uint_as_float(u.w);
    f[4] = __uint_as_float(w.x); f[5] = __uint_as_float(w.y); f[6] = __uint_as_float(w.z); f[7] = __uint_as_float(w.w);
    return;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) f[i] = (float)p[i];
}
template <typename T> __device__ __forceinline__ void store8(T* p, bool vec, const float* f) {
  if constexpr (sizeof(T) == 2) {
    if (vec) {
      *reinterpret_cast<uint4*>(p) = pack8(f);
      return;
    }
  } else if (vec) {
    *reinterpret_cast<float4*>(p) = make_float4(f[0], f[1], f[2], f[3]);
    *reinterpret_cast<float4*>(p + 4) = make_float4(f[4], f[5], f[6], f[7]);
    return;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) p[i] = (T)f[i];
}

// max over the 1 << bits lanes of a group
__device__ __forceinline__ uint32_t group_max(uint32_t v, int bits) {
  for (int o = (1 << bits) >> 1; o > 0; o >>= 1) v = max(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}
__device__ __forceinline__ float group_sum(float v, int bits) {
  for (int o = (1 << bits) >> 1; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// A lane's eight codes, given the head's largest magnitude as bits, and the scale
template <bool INT8> __device__ __forceinline__ uint2 codes8(const float* x, uint32_t top, float& scale) {
  if (top >= 0x7f800000u) {                                        // an infinity or NaN is among them
    scale = __uint_as_float(0x7fc00000u);
    return make_uint2(0u, 0u);
  }
  const float a = fmaxf(__uint_as_float(top), LEAST);
  const int e = (int)(__float_as_uint(a) >> 23) - 127;             // a = 1.m 2^e, -100 <= e <= 127
  uint2 r;
  if constexpr (INT8) {
    scale = a / 127.f;
    // 127 x / a, correctly rounded (a quotient's estimate and one correction by its exact remainder), so that a tie is a tie: x = a / 2 is 63.5 whatever 1 / a rounds to.
    // Both sides are divided by 128 and by a power of two near a, which is exact and keeps 127 x and 1 / a among the normal numbers.
    const float down = __uint_as_float((uint32_t)(127 - min(e, 126)) << 23), as = a * down, y = __frcp_rn(as), f = down * (127.f / 128.f);
    uint32_t c[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float n = x[i] * f, q = n * y;
      c[i] = (uint32_t)__float2int_rn(fmaf(fmaf(-as, q, n), y, q) * 128.f);
    }
    r.x = __byte_perm(__byte_perm(c[0], c[1], 0x0040), __byte_perm(c[2], c[3], 0x0040), 0x5410);
    r.y = __byte_perm(__byte_perm(c[4], c[5], 0x0040), __byte_perm(c[6], c[7], 0x0040), 0x5410);
  } else {
    const int s = e - 8 + ((__float_as_uint(a) & 0x7fffffu) > 0x600000u);   // 448 = 1.75 * 2^8
    scale = __uint_as_float((uint32_t)(127 + s) << 23);
    const float inv = __uint_as_float((uint32_t)(127 - s) << 23);
    uint32_t c[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float2 y = make_float2(x[2 * i] * inv, x[2 * i + 1] * inv);
      if (s == 120) y = make_float2(fminf(fmaxf(y.x, -240.f), 240.f), fminf(fmaxf(y.y, -240.f), 240.f));   // (256 would read back as 2^128)
      c[i] = __nv_cvt_float2_to_fp8x2(y, __NV_SATFINITE, __NV_E4M3);
    }
    r.x = c[0] | c[1] << 16;
    r.y = c[2] | c[3] << 16;
  }
  return r;
}

struct Side {
  const void* x;                                                   // rows of activations (store) or where they go (load)
  long long ld;
  Cache8 c;
  int bits, vec, norm;                                             // lanes of a head as a power of two; rows are whole 16-byte vectors apart
};

// Grid: blocks of heads of k and, behind them, of v
template <typename T, bool INT8, int NV>
__global__ void __launch_bounds__(THREADS) kv_store_8bit_kernel(Side k, Side v, const int* __restrict__ meta, int M, int G, int k_blocks, float eps) {
  pdl_launch_dependents();
  pdl_wait();
  const bool is_v = (int)blockIdx.x >= k_blocks;
  const Side& s = is_v ? v : k;
  const int lane = threadIdx.x & ((1 << s.bits) - 1);
  const unsigned i = (is_v ? blockIdx.x - k_blocks : blockIdx.x) * (THREADS >> s.bits) + (threadIdx.x >> s.bits);
  const bool there = i < (unsigned)M * G;
  const int row = there ? i / (unsigned)G : 0, g = there ? i - row * G : 0;
  const int2 at = make_int2(meta[2ll * row], meta[2ll * row + 1]);
  const int vecs = s.c.dim >> 3;
  const T* src = reinterpret_cast<const T*>(s.x) + row * s.ld + g * s.c.dim;
  float x[NV][8];
  uint32_t top = 0u;
  float ss = 0.f;
#pragma unroll
  for (int n = 0; n < NV; ++n) {
    const int c = lane + (n << s.bits);
    if (there && c < vecs) {
      load8(src + c * 8, s.vec, x[n]);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) x[n][j] = 0.f;
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) ss = fmaf(x[n][j], x[n][j], ss);
  }
  if (s.norm) {
    const float inv = 1.f / sqrtf(group_sum(ss, s.bits) / (float)s.c.dim + eps);
#pragma unroll
    for (int n = 0; n < NV; ++n)
#pragma unroll
      for (int j = 0; j < 8; ++j) x[n][j] *= inv;
  }
#pragma unroll
  for (int n = 0; n < NV; ++n)
#pragma unroll
    for (int j = 0; j < 8; ++j) top = max(top, __float_as_uint(x[n][j]) & 0x7fffffffu);     // (as whole numbers: NaN above infinity above the rest)
  top = group_max(top, s.bits);
  if (!there || !s.c.holds(at.x, at.y)) return;
  uint8_t* dst = s.c.at(at.x, at.y, g);
  float scale;
#pragma unroll
  for (int n = 0; n < NV; ++n) {
    const int c = lane + (n << s.bits);
    const uint2 r = codes8<INT8>(x[n], top, scale);
    if (c < vecs) *reinterpret_cast<uint2*>(dst + c * 8) = r;
  }
  if (lane == 0) s.c.scale_at(at.x, g)[at.y] = scale;
}

template <bool INT8> __device__ __forceinline__ void numbers8(const uint2& u, float scale, float* f) {
  const uint32_t w[2] = {u.x, u.y};
#pragma unroll
  for (int h = 0; h < 2; ++h)
#pragma unroll
    for (int j = 0; j < 4; j += 2) {
      float2 y;
      if constexpr (INT8) {
        y = make_float2((float)(int8_t)(w[h] >> (8 * j)), (float)(int8_t)(w[h] >> (8 * j + 8)));
      } else {
        const __half2_raw r = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w[h] >> (8 * j)), __NV_E4M3);
        y = __half22float2(__half2(r));
      }
      f[4 * h + j] = y.x * scale;
      f[4 * h + j + 1] = y.y * scale;
    }
}

template <typename T, bool INT8>
__global__ void __launch_bounds__(THREADS) kv_load_8bit_kernel(Side k, Side v, const int* __restrict__ meta, int M, int G, int k_blocks) {
  pdl_launch_dependents();
  pdl_wait();
  const bool is_v = (int)blockIdx.x >= k_blocks;
  const Side& s = is_v ? v : k;
  const int lane = threadIdx.x & ((1 << s.bits) - 1);
  const unsigned i = (is_v ? blockIdx.x - k_blocks : blockIdx.x) * (THREADS >> s.bits) + (threadIdx.x >> s.bits);
  if (i >= (unsigned)M * G) return;
  const int row = i / (unsigned)G, g = i - row * G;
  const int2 at = make_int2(meta[2ll * row], meta[2ll * row + 1]);
  T* dst = reinterpret_cast<T*>(const_cast<void*>(s.x)) + row * s.ld + g * s.c.dim;
  const bool held = s.c.holds(at.x, at.y);
  const uint8_t* src = held ? s.c.at(at.x, at.y, g) : nullptr;
  const float scale = held ? s.c.scale_at(at.x, g)[at.y] : __uint_as_float(0x7fc00000u);
  for (int c = lane; c < s.c.dim >> 3; c += 1 << s.bits) {
    float f[8];
    numbers8<INT8>(held ? *reinterpret_cast<const uint2*>(src + c * 8) : make_uint2(0u, 0u), scale, f);
    store8(dst + c * 8, s.vec, f);
  }
}

Side make_side(const void* x, long long ld, int act_f32, const LiaCacheView* view, int norm) {
  Side s{x, ld, cache8(view), 0, 0, norm};
  const int vecs = view->dim / 8;
  while ((1 << s.bits) < vecs && s.bits < 5) ++s.bits;
  const int per = act_f32 ? 4 : 8;
  s.vec = reinterpret_cast<uintptr_t>(x) % 16 == 0 && ld % per == 0;
  return s;
}

const char* sides_wrong(const void* k, const void* v, const void* meta, const LiaCacheView* kc, const LiaCacheView* vc, long long ldk, long long ldv, int M, int G) {
  const char* w = nullptr;
  if (!k || !v || !meta || M < 0 || G <= 0) return "null pointer or no heads";
  if ((w = cache8_wrong(kc, 8)) || (w = cache8_wrong(vc, 8))) return w;
  if (kc->type == LIA_CACHE_BF16 || kc->type != vc->type) return "both caches have to be int8, or both e4m3";
  if (kc->slots != vc->slots || kc->capacity != vc->capacity) return "caches of different sizes";
  if (kc->dim % 8 || vc->dim % 8 || kc->dim > 1024 || vc->dim > 1024) return "heads have to be multiples of 8 channels, 1024 at most";
  if ((long long)M * G >= 1ll << 31) return "too many rows";
  if (ldk < (long long)G * kc->dim || ldv < (long long)G * vc->dim) return "rows shorter than their heads";
  return w;
}

long long head_blocks(const Side& s, int M, int G) { return (((long long)M * G << s.bits) + THREADS - 1) / THREADS; }   // (at most 2^28)

}  // namespace

extern "C" int lia_kv_store_8bit(const void* k, long long ldk, const void* v, long long ldv, int act_f32, const int* meta, const LiaCacheView* kc, const LiaCacheView* vc, int M, int G,
                                 float eps, int norm_values, lia_stream_t stream) {
  const char* wrong = sides_wrong(k, v, meta, kc, vc, ldk, ldv, M, G);
  LIA_CHECK_ARG(!wrong, "lia_kv_store_8bit: %s", wrong);
  if (M == 0) return LIA_OK;
  const Side a = make_side(k, ldk, act_f32, kc, 0), b = make_side(v, ldv, act_f32, vc, norm_values != 0);
  const long long ka = head_blocks(a, M, G), blocks = ka + head_blocks(b, M, G);
  const int widest = kc->dim > vc->dim ? kc->dim : vc->dim;
  auto go = [&](auto kernel) {
    return lia_launch(kernel, dim3((unsigned)blocks), dim3(THREADS), 0, reinterpret_cast<cudaStream_t>(stream), a, b, meta, M, G, (int)ka, eps);
  };
  const bool i8 = kc->type == LIA_CACHE_INT8;
  if (widest <= 256) {                                             // one vector a lane
    if (act_f32) LIA_CUDA(i8 ? go(kv_store_8bit_kernel<float, true, 1>) : go(kv_store_8bit_kernel<float, false, 1>));
    else LIA_CUDA(i8 ? go(kv_store_8bit_kernel<bf16, true, 1>) : go(kv_store_8bit_kernel<bf16, false, 1>));
  } else {
    if (act_f32) LIA_CUDA(i8 ? go(kv_store_8bit_kernel<float, true, 4>) : go(kv_store_8bit_kernel<float, false, 4>));
    else LIA_CUDA(i8 ? go(kv_store_8bit_kernel<bf16, true, 4>) : go(kv_store_8bit_kernel<bf16, false, 4>));
  }
  return LIA_OK;
}

extern "C" int lia_kv_load_8bit(const int* meta, const LiaCacheView* kc, const LiaCacheView* vc, void* k, long long ldk, void* v, long long ldv, int out_f32, int M, int G,
                                lia_stream_t stream) {
  const char* wrong = sides_wrong(k, v, meta, kc, vc, ldk, ldv, M, G);
  LIA_CHECK_ARG(!wrong, "lia_kv_load_8bit: %s", wrong);
  if (M == 0) return LIA_OK;
  const Side a = make_side(k, ldk, out_f32, kc, 0), b = make_side(v, ldv, out_f32, vc, 0);
  const long long ka = head_blocks(a, M, G), blocks = ka + head_blocks(b, M, G);
  auto go = [&](auto kernel) {
    return lia_launch(kernel, dim3((unsigned)blocks), dim3(THREADS), 0, reinterpret_cast<cudaStream_t>(stream), a, b, meta, M, G, (int)ka);
  };
  const bool i8 = kc->type == LIA_CACHE_INT8;
  if (out_f32) LIA_CUDA(i8 ? go(kv_load_8bit_kernel<float, true>) : go(kv_load_8bit_kernel<float, false>));
  else LIA_CUDA(i8 ? go(kv_load_8bit_kernel<bf16, true>) : go(kv_load_8bit_kernel<bf16, false>));
  return LIA_OK;
}
