// Keys and values in 4 bits: quantised as they are written into a cache, and read back.
//
//   a = max |x| over 32 channels of a head of one token, s = bf16(a / 7), code = rint(x / s) in -7 .. 7, x stands for code * s: 4.5 bits a number
//
// An even grid without an offset: a group's zero is a zero, and a score is a sum of whole numbers times one scale.  Groups of 32: of normal numbers they leave 1 / 11 of their size as error, whole heads of
// 128 1 / 9, and a channel that is ten times the others takes the bits of 31 others instead of 127.
//
// Eight lanes have a head: lane q takes the channels 4 q .. 4 q + 3 of every group, which are 64 neighbouring bytes of bf16 activations for the eight, and whose codes are neighbours in the cache (byte4()).  Up
// to four groups at a time, so that a lane's codes of 128 channels are one 8-byte store; each lane sees to one group's scale, which the others get by shuffles.
//
// 7169 tokens with 8 heads of 128 (29 MB each of keys and values in, 8 MB out; ten calls in a graph): store 11.7 us, values normed 12.6, of fp32 numbers 14.7 and 14.2, bound by instructions (22 a number for 32
// lanes, 78 % of the issue slots; with 40 registers instead of 32 a thread half a microsecond more, every lane with all groups' scales 2.7); load 9.2, to fp32 10.0, instructions too (74 % of the issue slots, memory
// 8 %: results stay in L2; keys and values by the same lanes: 2.5 more, and the store 1.1).
#include "cache8.cuh"
#include "pairs.cuh"

namespace {

constexpr int THREADS = 256, LANES = 8, AT_ONCE = 4;               // lanes of a head, groups that a lane takes at a time
constexpr float LEAST = 7.888609052210118e-31f;                    // 2^-100: keeps scales and their inverses normal numbers

struct Side {
  const void* x;                                                   // rows of activations (store) or where they go (load)
  long long ld;
  Cache8 c;
  int vec, norm;                                                   // rows' fours are whole vectors apart
};
struct Head {
  bool there;
  int row, g, q, slot, pos;
};
__device__ __forceinline__ Head head_of(unsigned block, const int* meta, int M, int G) {
  Head h;
  const unsigned i = block * (THREADS / LANES) + threadIdx.x / LANES;
  h.there = i < (unsigned)M * G;
  h.row = h.there ? i / (unsigned)G : 0;
  h.g = h.there ? i - h.row * (unsigned)G : 0;
  h.q = threadIdx.x % LANES;
  h.slot = h.there ? meta[2ll * h.row] : -1;
  h.pos = h.there ? meta[2ll * h.row + 1] : -1;
  return h;
}

// Four numbers as they come
template <typename T> struct Raw4 {
  uint32_t w[sizeof(T)];
};
template <typename T> __device__ __forceinline__ Raw4<T> load4(const T* p, bool vec) {
  Raw4<T> r;
  if (vec) {
    if constexpr (sizeof(T) == 2) *reinterpret_cast<uint2*>(r.w) = __ldcg(reinterpret_cast<const uint2*>(p));
    else *reinterpret_cast<uint4*>(r.w) = ldg_act(p);
  } else {
    T t[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) t[i] = p[i];
#pragma unroll
    for (int i = 0; i < (int)sizeof(T); ++i) r.w[i] = reinterpret_cast<const uint32_t*>(t)[i];
  }
  return r;
}
template <typename T> __device__ __forceinline__ void numbers_of(const Raw4<T>& r, float* x) {
  if constexpr (sizeof(T) == 2) {
    unpack_bf16x2(r.w[0], x[0], x[1]);
    unpack_bf16x2(r.w[1], x[2], x[3]);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = __uint_as_float(r.w[i]);
  }
}
// Of the four groups' largest magnitudes, each over the eight lanes of a head, the bits of that of group 2 (q / 4) + q % 2 (as whole numbers NaN is above infinity and that above the rest)
__device__ __forceinline__ int group_of(int q) { return (q >> 2) * 2 + (q & 1); }
__device__ __forceinline__ int lane_of(int g) { return (g >> 1) * 4 + (g & 1); }
template <typename T> __device__ __forceinline__ uint32_t most_of(const Raw4<T>* raw, int q) {
  const bool last = q & 4, odd = q & 1;                            // halves of the lanes give each other what they do not keep
  if constexpr (sizeof(T) == 2) {                                  // two groups of 16 bits at a time
    uint32_t m[AT_ONCE], two[2];
#pragma unroll
    for (int g = 0; g < AT_ONCE; ++g) m[g] = __vmaxu2(raw[g].w[0] & 0x7fff7fffu, raw[g].w[1] & 0x7fff7fffu);
#pragma unroll
    for (int g = 0; g < 2; ++g) two[g] = __vmaxu2(__byte_perm(m[2 * g], m[2 * g + 1], 0x5410), __byte_perm(m[2 * g], m[2 * g + 1], 0x7632));
    uint32_t mine = __vmaxu2(last ? two[1] : two[0], __shfl_xor_sync(0xffffffffu, last ? two[0] : two[1], 4));
    mine = __vmaxu2(mine, __shfl_xor_sync(0xffffffffu, mine, 2));
    mine = __vmaxu2(mine, __shfl_xor_sync(0xffffffffu, mine, 1));
    return odd ? mine & 0xffff0000u : mine << 16;
  } else {
    uint32_t m[AT_ONCE];
#pragma unroll
    for (int g = 0; g < AT_ONCE; ++g) {
      m[g] = 0u;
#pragma unroll
      for (int i = 0; i < 4; ++i) m[g] = max(m[g], raw[g].w[i] & 0x7fffffffu);
    }
    const uint32_t even_group = max(last ? m[2] : m[0], __shfl_xor_sync(0xffffffffu, last ? m[0] : m[2], 4)), odd_group = max(last ? m[3] : m[1], __shfl_xor_sync(0xffffffffu, last ? m[1] : m[3], 4));
    uint32_t mine = max(odd ? odd_group : even_group, __shfl_xor_sync(0xffffffffu, odd ? even_group : odd_group, 1));
    return max(mine, __shfl_xor_sync(0xffffffffu, mine, 2));
  }
}
template <typename T> __device__ __forceinline__ void store4(T* p, bool vec, const float* x) {
  if constexpr (sizeof(T) == 2) {
    if (vec) {
      *reinterpret_cast<uint2*>(p) = make_uint2(pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]));
      return;
    }
  } else if (vec) {
    *reinterpret_cast<float4*>(p) = *reinterpret_cast<const float4*>(x);
    return;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) p[i] = (T)x[i];
}

// x / d, correctly rounded, with inv = 1 / d correctly rounded (Markstein 1990: the estimate and one correction by its exact remainder)
__device__ __forceinline__ float quotient(float x, float d, float inv) {
  const float q = x * inv;
  return fmaf(fmaf(-d, q, x), inv, q);
}

// 1 / d of a number of 8 bits, correctly rounded (an inverse of 8 bits is further than 2^-33 of itself from a border between numbers of 24)
__device__ __forceinline__ float inverse(float d) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(d));
  return fmaf(fmaf(-d, y, 1.f), y, y);
}

// `n` numbers of 16 bits, as wide as a lane's n groups of ng lie; eight lanes' are neighbours
__device__ __forceinline__ void put_units(uint16_t* dst, int ng, int n, const uint32_t* u) {
  if ((ng & 3) == 0) {
    *reinterpret_cast<uint2*>(dst) = make_uint2(u[0] | u[1] << 16, u[2] | u[3] << 16);
  } else if ((ng & 1) == 0) {
    *reinterpret_cast<uint32_t*>(dst) = u[0] | u[1] << 16;
    if (n > 2) *reinterpret_cast<uint32_t*>(dst + 2) = u[2] | u[3] << 16;
  } else {
#pragma unroll
    for (int i = 0; i < AT_ONCE; ++i)
      if (i < n) dst[i] = (uint16_t)u[i];
  }
}
__device__ __forceinline__ void get_units(const uint16_t* src, int ng, int n, uint32_t* u) {
  if ((ng & 3) == 0) {
    const uint2 w = __ldcg(reinterpret_cast<const uint2*>(src));
    u[0] = w.x & 0xffffu, u[1] = w.x >> 16, u[2] = w.y & 0xffffu, u[3] = w.y >> 16;
  } else if ((ng & 1) == 0) {
    const uint32_t a = __ldcg(reinterpret_cast<const uint32_t*>(src)), b = n > 2 ? __ldcg(reinterpret_cast<const uint32_t*>(src + 2)) : 0u;
    u[0] = a & 0xffffu, u[1] = a >> 16, u[2] = b & 0xffffu, u[3] = b >> 16;
  } else {
#pragma unroll
    for (int i = 0; i < AT_ONCE; ++i) u[i] = i < n ? __ldcg(src + i) : 0u;
  }
}

constexpr float ROUND = 12582912.f;                                // 1.5 * 2^23: what is added to it is rounded to a whole number

// Normed numbers' codes are of x (1 / root) (1 / scale), each rounded to 24 bits: a code may be the neighbour's where the quotient is within some 2^-22 of itself from a border, as it may for the root, whose sum of
// squares is rounded.  Of 7.3 million codes as many differ from those of 64 bits as with divisions rounded correctly, none to two, which take 13.2 us instead of 12.2 (with ties told apart 14.9).

template <typename T> __device__ __forceinline__ void store_heads(const Side& s, bool norm, const Head& h, float eps) {
  const int ng = s.c.dim / GROUP4;
  const T* src = reinterpret_cast<const T*>(s.x) + h.row * s.ld + h.g * s.c.dim + h.q * 4;
  Raw4<T> raw[AT_ONCE];
  auto load = [&](int g0) {
    const int n = h.there ? ng - g0 : 0;
    if (s.vec && n >= AT_ONCE) {
#pragma unroll
      for (int g = 0; g < AT_ONCE; ++g) raw[g] = load4(src + (g0 + g) * GROUP4, true);
    } else {
#pragma unroll
      for (int g = 0; g < AT_ONCE; ++g) raw[g] = g < n ? load4(src + (g0 + g) * GROUP4, s.vec) : Raw4<T>{};
    }
  };
  load(0);
  float root = 1.f, inv_root = 1.f;
  if (norm) {
    float sum = 0.f;
    for (int g0 = 0; g0 < ng; g0 += AT_ONCE) {
      if (g0 > 0) load(g0);
      float part[AT_ONCE];
#pragma unroll
      for (int g = 0; g < AT_ONCE; ++g) {
        float x[4];
        numbers_of(raw[g], x);
        part[g] = fmaf(x[0], x[0], x[1] * x[1]) + fmaf(x[2], x[2], x[3] * x[3]);
      }
      sum += (part[0] + part[1]) + (part[2] + part[3]);
    }
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    root = sqrtf(sum / (float)s.c.dim + eps);
    inv_root = 1.f / root;
    if (root > 3.402823466e38f) root = 0.f;                        // (quotients are 0, and stay so)
    if (ng > AT_ONCE) load(0);
  }
  const bool held = s.c.holds(h.slot, h.pos);
  uint16_t* codes = held ? reinterpret_cast<uint16_t*>(s.c.at(h.slot, h.pos, h.g)) + h.q * ng : nullptr;
  uint16_t* scales = held ? reinterpret_cast<uint16_t*>(s.c.scale4_at(h.slot, h.g)) + (long long)h.pos * ng : nullptr;
  for (int g0 = 0; g0 < ng; g0 += AT_ONCE) {
    if (g0 > 0) load(g0);
    // a lane sees to one group's scale (two lanes to the same), which the others get from it
    float a = __uint_as_float(most_of(raw, h.q));
    if (norm) a = quotient(a, root, inv_root);                   // (the largest before, divided as it is: rounding keeps order)
    const bool bad = !(a <= 3.402823466e38f);
    const __nv_bfloat16 s16 = __float2bfloat16_rn(quotient(fmaxf(a, LEAST), 7.f, 1.f / 7.f));
    const float scale = __bfloat162float(s16);
    const float inv = bad ? 0.f : inverse(scale);
    uint32_t units[AT_ONCE];
#pragma unroll
    for (int g = 0; g < AT_ONCE; ++g) {
      const float by = __shfl_sync(0xffffffffu, inv, lane_of(g), LANES), d = __shfl_sync(0xffffffffu, scale, lane_of(g), LANES);
      float x[4], c[4];                                            // codes + ROUND, whose lowest bits are the codes
      numbers_of(raw[g], x);
#pragma unroll
      for (int i = 0; i < 4; i += 2) {
        const f32x2 y = pack2(x[i], x[i + 1]);
        if (norm) {                                                // (one after the other: the two inverses' product may be infinite)
          unpack2(fma2(mul2(y, both(inv_root)), both(by), both(ROUND)), c[i], c[i + 1]);
        } else {
          const f32x2 e = mul2(y, both(by));
          unpack2(add2(fma2(fma2(both(-d), e, y), both(by), e), both(ROUND)), c[i], c[i + 1]);   // (quotient())
        }
      }
      // where rounding the quotient to 24 bits made a tie of it, the exact rest (a code times 8 bits) tells on which side it was; of two numbers of 8 bits it is a tie or far from one
      if (sizeof(T) == 4 && !norm) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float rest = fmaf(-(c[i] - ROUND), d, x[i]);
          c[i] += fabsf(rest) > 0.5f * d ? copysignf(1.f, rest) : 0.f;
        }
      }
      uint32_t u = 0x8888u;                                        // four codes + 8
#pragma unroll
      for (int i = 0; i < 4; ++i) u += __float_as_uint(c[i]) << (4 * i);
      units[g] = by == 0.f ? 0x8888u : u & 0xffffu;
    }
    if (!held) continue;
    const int n = min(AT_ONCE, ng - g0), own = group_of(h.q);
    put_units(codes + g0, ng, n, units);
    if ((h.q & 2) == 0 && own < n) scales[g0 + own] = bad ? 0x7fc0u : __bfloat16_as_ushort(s16);
  }
}

// Grid: blocks of heads of k and, behind them, of v (each with code of its own: which of two it is costs a lookup for whatever is asked of it)
template <typename T>
__global__ void __launch_bounds__(THREADS, sizeof(T) == 2 ? 8 : 4) kv_store_4bit_kernel(const __grid_constant__ Side k, const __grid_constant__ Side v, const int* __restrict__ meta, int M, int G, int blocks, float eps) {
  pdl_launch_dependents();
  pdl_wait();
  if ((int)blockIdx.x < blocks) store_heads<T>(k, false, head_of(blockIdx.x, meta, M, G), eps);
  else store_heads<T>(v, v.norm, head_of(blockIdx.x - blocks, meta, M, G), eps);
}

template <typename T> __device__ __forceinline__ void load_heads(const Side& s, const Head& h) {
  if (!h.there) return;
  const int ng = s.c.dim / GROUP4;
  const bool held = s.c.holds(h.slot, h.pos);
  const uint16_t* codes = held ? reinterpret_cast<const uint16_t*>(s.c.at(h.slot, h.pos, h.g)) + h.q * ng : nullptr;
  const uint16_t* scales = held ? reinterpret_cast<const uint16_t*>(s.c.scale4_at(h.slot, h.g)) + (long long)h.pos * ng : nullptr;
  T* dst = reinterpret_cast<T*>(const_cast<void*>(s.x)) + h.row * s.ld + h.g * s.c.dim + h.q * 4;
  for (int g0 = 0; g0 < ng; g0 += AT_ONCE) {
    const int n = min(AT_ONCE, ng - g0);
    uint32_t u[AT_ONCE] = {}, sc[AT_ONCE] = {0x7fc0u, 0x7fc0u, 0x7fc0u, 0x7fc0u};
    if (held) {
      get_units(codes + g0, ng, n, u);
      get_units(scales + g0, ng, n, sc);
    }
#pragma unroll
    for (int g = 0; g < AT_ONCE; g += 2) {                         // two groups' codes at a time, as 128 + n in bf16; a code times a scale has 12 bits, which are rounded once
      const uint32_t two = u[g] | u[g + 1] << 16;
      __nv_bfloat162 c[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t w = (two >> (4 * i) & 0x000f000fu) | 0x43004300u;
        c[i] = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&w), __float2bfloat162_rn(136.f));
      }
#pragma unroll
      for (int o = 0; o < 2; ++o) {
        if (g + o >= n) break;
        const float scale = __uint_as_float(sc[g + o] << 16);
        float x[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = (o ? __high2float(c[i]) : __low2float(c[i])) * scale;
        store4(dst + (g0 + g + o) * GROUP4, s.vec, x);
      }
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(THREADS) kv_load_4bit_kernel(const __grid_constant__ Side k, const __grid_constant__ Side v, const int* __restrict__ meta, int M, int G, int blocks) {
  pdl_launch_dependents();
  pdl_wait();
  if ((int)blockIdx.x < blocks) load_heads<T>(k, head_of(blockIdx.x, meta, M, G));
  else load_heads<T>(v, head_of(blockIdx.x - blocks, meta, M, G));
}

Side make_side(const void* x, long long ld, int act_f32, const LiaCacheView* view, int norm) {
  const int bytes = act_f32 ? 16 : 8;
  return {x, ld, cache8(view), reinterpret_cast<uintptr_t>(x) % bytes == 0 && ld % 4 == 0, norm};
}

const char* sides_wrong(const void* k, const void* v, const void* meta, const LiaCacheView* kc, const LiaCacheView* vc, long long ldk, long long ldv, int M, int G) {
  const char* w = nullptr;
  if (M < 0 || G <= 0 || (M > 0 && (!k || !v || !meta))) return "null pointer or no heads";     // (no rows have no address)
  if ((w = cache8_wrong(kc, 8)) || (w = cache8_wrong(vc, 8))) return w;
  if (kc->type != LIA_CACHE_INT4 || vc->type != LIA_CACHE_INT4) return "both caches have to be of 4 bits";
  if (kc->slots != vc->slots || kc->capacity != vc->capacity) return "caches of different sizes";
  if (kc->dim > 1024 || vc->dim > 1024) return "heads have 1024 channels at most";
  if ((long long)M * G >= 1ll << 31) return "too many rows";
  if (ldk < (long long)G * kc->dim || ldv < (long long)G * vc->dim) return "rows shorter than their heads";
  return w;
}

}  // namespace

extern "C" int lia_kv_store_4bit(const void* k, long long ldk, const void* v, long long ldv, int act_f32, const int* meta, const LiaCacheView* kc, const LiaCacheView* vc, int M, int G,
                                 float eps, int norm_values, lia_stream_t stream_) {
  const char* wrong = sides_wrong(k, v, meta, kc, vc, ldk, ldv, M, G);
  LIA_CHECK_ARG(!wrong, "lia_kv_store_4bit: %s", wrong);
  if (M == 0) return LIA_OK;
  const Side a = make_side(k, ldk, act_f32, kc, 0), b = make_side(v, ldv, act_f32, vc, norm_values != 0);
  const int blocks = (int)(((long long)M * G * LANES + THREADS - 1) / THREADS);
  cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_);
  if (act_f32) LIA_CUDA(lia_launch(kv_store_4bit_kernel<float>, dim3(2 * blocks), dim3(THREADS), 0, stream, a, b, meta, M, G, blocks, eps));
  else LIA_CUDA(lia_launch(kv_store_4bit_kernel<bf16>, dim3(2 * blocks), dim3(THREADS), 0, stream, a, b, meta, M, G, blocks, eps));
  return LIA_OK;
}

extern "C" int lia_kv_load_4bit(const int* meta, const LiaCacheView* kc, const LiaCacheView* vc, void* k, long long ldk, void* v, long long ldv, int out_f32, int M, int G,
                                lia_stream_t stream_) {
  const char* wrong = sides_wrong(k, v, meta, kc, vc, ldk, ldv, M, G);
  LIA_CHECK_ARG(!wrong, "lia_kv_load_4bit: %s", wrong);
  if (M == 0) return LIA_OK;
  const Side a = make_side(k, ldk, out_f32, kc, 0), b = make_side(v, ldv, out_f32, vc, 0);
  const int blocks = (int)(((long long)M * G * LANES + THREADS - 1) / THREADS);
  cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_);
  if (out_f32) LIA_CUDA(lia_launch(kv_load_4bit_kernel<float>, dim3(2 * blocks), dim3(THREADS), 0, stream, a, b, meta, M, G, blocks));
  else LIA_CUDA(lia_launch(kv_load_4bit_kernel<bf16>, dim3(2 * blocks), dim3(THREADS), 0, stream, a, b, meta, M, G, blocks));
  return LIA_OK;
}
