// Keys and values in 8 bits: quantised as they are written into a cache, and read back.
//
//   int8   a = max |x| over a head of one token, scale = a / 127, code = rint(127 x / a): an even grid, for heads whose numbers are alike
//   e4m3   scale = 2^e, the least with a / 2^e <= 448, code = x / 2^e rounded to 4 significant bits.  A float keeps its 4 bits at any of 15 powers of two, so a power of two
//          loses nothing against a / 448 down to a / 28672, and makes scaling and reading back exact.
// One scale for each head of each token: a token that comes later changes nothing that is there, and attention multiplies scores and weights by scales instead of channels by them.
//
// Both kernels move each number once.  A lane has 32 neighbouring channels of a head (four lanes a head of 128), which divides the addresses, the scale and the steps of finding the largest magnitude
// among them.  Magnitudes of bf16 numbers are compared as pairs of whole numbers, and a normed head's largest is the largest before, divided as it is, because rounding keeps order.
//
// What bounds them, by counters: storing normed values instructions, some 25 issued a number (7169 tokens of 8 heads of 128 to e4m3 11.5 us, issue slots 71 % busy, memory 25 %); reading back the SMs' own
// way to memory (86 % of its peak, memory 49 %: 16 histories of 8191 tokens 136 us): a lane's vectors are neighbours, so that one instruction of a warp touches 16 bytes of every 64, half of
// each sector.
#include <cuda_fp8.h>

#include "cache8.cuh"

namespace {

constexpr int THREADS = 256;
constexpr float LEAST = 7.888609052210118e-31f;                    // 2^-100: keeps scales and their inverses normal numbers

// Eight numbers as they come: one or two 16-byte vectors
template <typename T> struct Raw8 {
  uint4 u[sizeof(T) / 2];
};
template <typename T> __device__ __forceinline__ Raw8<T> load8(const T* p, bool vec) {
  Raw8<T> r;
  if (vec) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) r.u[i] = ldg_act(p + 8 / (sizeof(T) / 2) * i);
  } else {
    T t[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) t[i] = p[i];
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) r.u[i] = reinterpret_cast<const uint4*>(t)[i];
  }
  return r;
}
template <typename T> __device__ __forceinline__ void numbers_of(const Raw8<T>& r, float* f) {
  if constexpr (sizeof(T) == 2) {
    unpack8(r.u[0], f);
  } else {
    f[0] = __uint_as_float(r.u[0].x); f[1] = __uint_as_float(r.u[0].y); f[2] = __uint_as_float(r.u[0].z); f[3] = __uint_as_float(r.u[0].w);
    f[4] = __uint_as_float(r.u[1].x); f[5] = __uint_as_float(r.u[1].y); f[6] = __uint_as_float(r.u[1].z); f[7] = __uint_as_float(r.u[1].w);
  }
}
// The largest magnitude's bits: of fp32 numbers, or of bf16 ones in both halves (as whole numbers NaN is above infinity and that above the rest)
template <typename T> __device__ __forceinline__ uint32_t most_of(const Raw8<T>& r, uint32_t m) {
#pragma unroll
  for (int i = 0; i < (int)sizeof(T) / 2; ++i) {
    const uint32_t w[4] = {r.u[i].x, r.u[i].y, r.u[i].z, r.u[i].w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if constexpr (sizeof(T) == 2) m = __vmaxu2(m, w[j] & 0x7fff7fffu);
      else m = max(m, w[j] & 0x7fffffffu);
    }
  }
  return m;
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

// How a head's numbers become codes, by its largest magnitude
template <bool INT8> struct Coder {
  float scale, f, y, as;                                           // scale NaN: codes are 0
  bool last;
  __device__ __forceinline__ explicit Coder(float largest) {
    if (!(largest <= 3.402823466e38f)) {                           // an infinity or NaN is among them
      scale = __uint_as_float(0x7fc00000u);
      f = y = as = 0.f;
      last = false;
      return;
    }
    const float a = fmaxf(largest, LEAST);
    const int e = (int)(__float_as_uint(a) >> 23) - 127;           // a = 1.m 2^e, -100 <= e <= 127
    if constexpr (INT8) {
      // 127 x / a, correctly rounded by Markstein's method (1990: an estimate of the quotient from the rounded reciprocal, and one correction by its exact remainder), so that a tie is a tie: x = a / 2
      // is 63.5 whatever 1 / a rounds to.  Both sides are divided by 128 and by a power of two near a, which keeps 127 x and 1 / a among the normal numbers.  127 x is exact for bf16 numbers; of fp32 ones it is
      // rounded once before, so that a code may be the neighbour's where the exact quotient is within 2^-23 of itself from a border.
      const float down = __uint_as_float((uint32_t)(127 - min(e, 126)) << 23);
      scale = a / 127.f;
      as = a * down;
      y = __frcp_rn(as);
      f = down * (127.f / 128.f);
      last = false;
    } else {
      const int s = e - 8 + ((__float_as_uint(a) & 0x7fffffu) > 0x600000u);            // 448 = 1.75 * 2^8
      scale = __uint_as_float((uint32_t)(127 + s) << 23);
      f = __uint_as_float((uint32_t)(127 - s) << 23);
      last = s == 120;
    }
  }
  __device__ __forceinline__ uint2 operator()(const float* x) const {
    uint32_t c[8];
    if constexpr (INT8) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {                                // (the sum's lowest bits are the rounded number: as = 0 gives 0)
        const float n = x[i] * f, q = n * y;
        c[i] = __float_as_uint(fmaf(fmaf(fmaf(-as, q, n), y, q), 128.f, 12582912.f));
      }
      if (as == 0.f) return make_uint2(0u, 0u);
      return make_uint2(__byte_perm(__byte_perm(c[0], c[1], 0x0040), __byte_perm(c[2], c[3], 0x0040), 0x5410),
                        __byte_perm(__byte_perm(c[4], c[5], 0x0040), __byte_perm(c[6], c[7], 0x0040), 0x5410));
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float2 t = make_float2(x[2 * i] * f, x[2 * i + 1] * f);
        if (last) t = make_float2(fminf(fmaxf(t.x, -240.f), 240.f), fminf(fmaxf(t.y, -240.f), 240.f));   // (256 would read back as 2^128)
        c[i] = __nv_cvt_float2_to_fp8x2(t, __NV_SATFINITE, __NV_E4M3);
      }
      if (f == 0.f) return make_uint2(0u, 0u);
      return make_uint2(c[0] | c[1] << 16, c[2] | c[3] << 16);
    }
  }
};

// x / root, with inv = 1 / root, by the same method.  (x * inv behind squares summed in one chain moved more normed values across a border between codes: the
// codes of 8 million were off by 1.8e-4 of their size, root mean square, instead of 2e-5.)
__device__ __forceinline__ float quotient(float x, float root, float inv) {
  const float q = x * inv;
  return fmaf(fmaf(-root, q, x), inv, q);
}

constexpr int NV = 4;                                              // vectors of eight neighbouring channels of a lane

struct Side {
  const void* x;                                                   // rows of activations (store) or where they go (load)
  long long ld;
  Cache8 c;
  int bits, vec, wide, norm;                                       // lanes of a head as a power of two; rows, and codes, are whole 16-byte vectors apart
};
struct Head {
  bool there;
  int row, g, lane, slot, pos;                                     // lane: of the head's
};
__device__ __forceinline__ Head head_of(const Side& s, int block, const int* meta, int M, int G) {
  Head h;
  const unsigned i = block * (THREADS >> s.bits) + (threadIdx.x >> s.bits);
  h.there = i < (unsigned)M * G;
  h.row = h.there ? i / (unsigned)G : 0;
  h.g = h.there ? i - h.row * (unsigned)G : 0;
  h.lane = threadIdx.x & ((1 << s.bits) - 1);
  h.slot = h.there ? meta[2ll * h.row] : -1;
  h.pos = h.there ? meta[2ll * h.row + 1] : -1;
  return h;
}

// Grid: blocks of heads of k and, behind them, of v
template <typename T, bool INT8>
__global__ void __launch_bounds__(THREADS) kv_store_8bit_kernel(Side k, Side v, const int* __restrict__ meta, int M, int G, int k_blocks, float eps) {
  pdl_launch_dependents();
  pdl_wait();
  const bool is_v = (int)blockIdx.x >= k_blocks;
  const Side& s = is_v ? v : k;
  const Head h = head_of(s, is_v ? blockIdx.x - k_blocks : blockIdx.x, meta, M, G);
  const int vecs = s.c.dim >> 3, c0 = h.lane * NV;
  const T* src = reinterpret_cast<const T*>(s.x) + h.row * s.ld + h.g * s.c.dim + c0 * 8;
  Raw8<T> raw[NV];
#pragma unroll
  for (int n = 0; n < NV; ++n) {
    if (h.there && c0 + n < vecs) raw[n] = load8(src + n * 8, s.vec);
    else raw[n] = Raw8<T>{};
  }
  uint32_t most = 0u;
#pragma unroll
  for (int n = 0; n < NV; ++n) most = most_of(raw[n], most);
  for (int o = (1 << s.bits) >> 1; o > 0; o >>= 1) {
    const uint32_t m = __shfl_xor_sync(0xffffffffu, most, o);
    most = sizeof(T) == 2 ? __vmaxu2(most, m) : max(most, m);
  }
  float largest = __uint_as_float(sizeof(T) == 2 ? max(most & 0xffffu, most >> 16) << 16 : most), inv = 1.f;
  float root = 1.f;
  if (s.norm) {
    float ss[NV] = {};
#pragma unroll
    for (int n = 0; n < NV; ++n) {
      float x[8];
      numbers_of(raw[n], x);
#pragma unroll
      for (int j = 0; j < 8; ++j) ss[n] = fmaf(x[j], x[j], ss[n]);
    }
    float sum = (ss[0] + ss[1]) + (ss[2] + ss[3]);
    for (int o = (1 << s.bits) >> 1; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    root = sqrtf(sum / (float)s.c.dim + eps);
    inv = 1.f / root;
    if (root > 3.402823466e38f) root = 0.f;                        // (quotients are 0, and stay so)
    largest = quotient(largest, root, inv);
  }
  if (!s.c.holds(h.slot, h.pos)) return;
  const Coder<INT8> code(largest);
  uint8_t* dst = s.c.at(h.slot, h.pos, h.g) + c0 * 8;
#pragma unroll
  for (int n = 0; n < NV; n += 2) {
    float x[8], y[8];
    numbers_of(raw[n], x);
    numbers_of(raw[n + 1], y);
    if (s.norm) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        x[j] = quotient(x[j], root, inv);
        y[j] = quotient(y[j], root, inv);
      }
    }
    const uint2 r = code(x), q = code(y);
    if (s.wide && c0 + n + 1 < vecs) {
      *reinterpret_cast<uint4*>(dst + n * 8) = make_uint4(r.x, r.y, q.x, q.y);
    } else {
      if (c0 + n < vecs) *reinterpret_cast<uint2*>(dst + n * 8) = r;
      if (c0 + n + 1 < vecs) *reinterpret_cast<uint2*>(dst + n * 8 + 8) = q;
    }
  }
  if (h.lane == 0) s.c.scale_at(h.slot, h.g)[h.pos] = code.scale;
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
  const Head h = head_of(s, is_v ? blockIdx.x - k_blocks : blockIdx.x, meta, M, G);
  if (!h.there) return;
  const int vecs = s.c.dim >> 3, c0 = h.lane * NV;
  const bool held = s.c.holds(h.slot, h.pos);
  const uint8_t* src = held ? s.c.at(h.slot, h.pos, h.g) + c0 * 8 : nullptr;
  const float scale = held ? __ldcg(s.c.scale_at(h.slot, h.g) + h.pos) : __uint_as_float(0x7fc00000u);
  uint2 codes[NV];
#pragma unroll
  for (int n = 0; n < NV; n += 2) {
    codes[n] = codes[n + 1] = make_uint2(0u, 0u);
    if (held && s.wide && c0 + n + 1 < vecs) {
      const uint4 u = ldg_act(src + n * 8);
      codes[n] = make_uint2(u.x, u.y);
      codes[n + 1] = make_uint2(u.z, u.w);
    } else if (held) {
      if (c0 + n < vecs) codes[n] = __ldcg(reinterpret_cast<const uint2*>(src + n * 8));
      if (c0 + n + 1 < vecs) codes[n + 1] = __ldcg(reinterpret_cast<const uint2*>(src + n * 8 + 8));
    }
  }
  T* dst = reinterpret_cast<T*>(const_cast<void*>(s.x)) + h.row * s.ld + h.g * s.c.dim + c0 * 8;
#pragma unroll
  for (int n = 0; n < NV; ++n) {
    float f[8];
    numbers8<INT8>(codes[n], scale, f);
    if (c0 + n < vecs) store8(dst + n * 8, s.vec, f);
  }
}

Side make_side(const void* x, long long ld, int act_f32, const LiaCacheView* view, int norm) {
  Side s{x, ld, cache8(view), 0, 0, 0, norm};
  while ((NV << s.bits) < view->dim / 8) ++s.bits;                 // (5 at most: 1024 channels)
  s.vec = reinterpret_cast<uintptr_t>(x) % 16 == 0 && ld % (act_f32 ? 4 : 8) == 0;
  s.wide = cache8_wrong(view, 16) == nullptr;
  return s;
}
int head_blocks(const Side& s, int M, int G) { return (int)((((long long)M * G << s.bits) + THREADS - 1) / THREADS); }

const char* sides_wrong(const void* k, const void* v, const void* meta, const LiaCacheView* kc, const LiaCacheView* vc, long long ldk, long long ldv, int M, int G) {
  const char* w = nullptr;
  if (M < 0 || G <= 0 || (M > 0 && (!k || !v || !meta))) return "null pointer or no heads";     // (no rows have no address)
  if ((w = cache8_wrong(kc, 8)) || (w = cache8_wrong(vc, 8))) return w;
  if (kc->type == LIA_CACHE_BF16 || kc->type != vc->type) return "both caches have to be int8, or both e4m3";
  if (kc->slots != vc->slots || kc->capacity != vc->capacity) return "caches of different sizes";
  if (kc->dim % 8 || vc->dim % 8 || kc->dim > 1024 || vc->dim > 1024) return "heads have to be multiples of 8 channels, 1024 at most";
  if ((long long)M * G >= 1ll << 31) return "too many rows";
  if (ldk < (long long)G * kc->dim || ldv < (long long)G * vc->dim) return "rows shorter than their heads";
  return w;
}

}  // namespace

extern "C" int lia_kv_store_8bit(const void* k, long long ldk, const void* v, long long ldv, int act_f32, const int* meta, const LiaCacheView* kc, const LiaCacheView* vc, int M, int G,
                                 float eps, int norm_values, lia_stream_t stream) {
  const char* wrong = sides_wrong(k, v, meta, kc, vc, ldk, ldv, M, G);
  LIA_CHECK_ARG(!wrong, "lia_kv_store_8bit: %s", wrong);
  if (M == 0) return LIA_OK;
  const Side a = make_side(k, ldk, act_f32, kc, 0), b = make_side(v, ldv, act_f32, vc, norm_values != 0);
  const int ka = head_blocks(a, M, G), blocks = ka + head_blocks(b, M, G);
  auto go = [&](auto kernel) { return lia_launch(kernel, dim3(blocks), dim3(THREADS), 0, reinterpret_cast<cudaStream_t>(stream), a, b, meta, M, G, ka, eps); };
  const bool i8 = kc->type == LIA_CACHE_INT8;
  if (act_f32) LIA_CUDA(i8 ? go(kv_store_8bit_kernel<float, true>) : go(kv_store_8bit_kernel<float, false>));
  else LIA_CUDA(i8 ? go(kv_store_8bit_kernel<bf16, true>) : go(kv_store_8bit_kernel<bf16, false>));
  return LIA_OK;
}

extern "C" int lia_kv_load_8bit(const int* meta, const LiaCacheView* kc, const LiaCacheView* vc, void* k, long long ldk, void* v, long long ldv, int out_f32, int M, int G,
                                lia_stream_t stream) {
  const char* wrong = sides_wrong(k, v, meta, kc, vc, ldk, ldv, M, G);
  LIA_CHECK_ARG(!wrong, "lia_kv_load_8bit: %s", wrong);
  if (M == 0) return LIA_OK;
  const Side a = make_side(k, ldk, out_f32, kc, 0), b = make_side(v, ldv, out_f32, vc, 0);
  const int ka = head_blocks(a, M, G), blocks = ka + head_blocks(b, M, G);
  auto go = [&](auto kernel) { return lia_launch(kernel, dim3(blocks), dim3(THREADS), 0, reinterpret_cast<cudaStream_t>(stream), a, b, meta, M, G, ka); };
  const bool i8 = kc->type == LIA_CACHE_INT8;
  if (out_f32) LIA_CUDA(i8 ? go(kv_load_8bit_kernel<float, true>) : go(kv_load_8bit_kernel<float, false>));
  else LIA_CUDA(i8 ? go(kv_load_8bit_kernel<bf16, true>) : go(kv_load_8bit_kernel<bf16, false>));
  return LIA_OK;
}
