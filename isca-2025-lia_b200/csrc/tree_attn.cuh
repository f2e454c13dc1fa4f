// What the kernels of attention of drafted tokens share (tree_attn.cu, tree_attn_sm100.cu): a portion, which keys its rows see, and rows that are formed key by key.
#pragma once
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "cache8.cuh"

namespace {

constexpr float LOG2E = 1.4426950408889634f;
// Values whose scale is below this count as if it were this, which puts them off by 2^-71 at most.  Their scores count all the same: a weight is p times the scale, relative to the largest such
// product, and with scales up to 2^29 a p of 2^-24 stays above the smallest normal number, from where it goes into the sum of the p.
constexpr float LEAST_SCALE = 0x1p-80f;

struct TreeArgs {
  const bf16* q;
  long long ldq;
  Cache8 k, v;
  const int* segs;                                                 // (whole numbers, wherever they lie)
  const unsigned long long* mask;
  int words;
  const int* depth;
  const float* temp;
  bf16* out;
  float* ws;                                                       // weighted values [splits][M * H][VDIM], then (maximum, sum of weights) [splits][M * H]
  int M, H, G, rep, rows, window, splits, tiles;
  float scale, softcap;
};

struct Portion {
  int slot, p0, row, n;
  bool held;                                                       // its slot, the rows, the mask and the launch have room for it
};
__device__ __forceinline__ Portion portion_of(const TreeArgs& a, int z) {
  const int* s = a.segs + 4ll * z;
  Portion p{s[0], s[1], s[2], s[3], true};
  p.held = (unsigned)p.slot < (unsigned)a.k.slots && p.p0 >= 0 && p.n >= 0 && p.n <= a.rows && p.row >= 0 && p.n <= a.M && p.row <= a.M - p.n && p.n <= a.k.capacity &&
           p.p0 <= a.k.capacity - p.n && (a.mask == nullptr || p.n <= 64 * a.words);
  return p;
}
// rows of a portion that is not held, as far as they are rows, by a block
template <int VDIM> __device__ __forceinline__ void nan_rows(const TreeArgs& a, const Portion& p) {
  const long long r0 = max(p.row, 0), r1 = min((long long)p.row + p.n, (long long)a.M), w = (long long)a.H * VDIM;
  for (long long i = r0 * w + threadIdx.x; i < r1 * w; i += blockDim.x) a.out[i] = __ushort_as_bfloat16((unsigned short)0x7fc0u);
}
__device__ __forceinline__ int depth_of(const TreeArgs& a, const Portion& p, int i) {
  return a.depth == nullptr ? i : min(max(a.depth[p.row + i], 0), 1 << 29);
}
// whether row i of a portion, `deep` behind its history, sees the key at position t < p0 + n
__device__ __forceinline__ bool sees(const TreeArgs& a, const Portion& p, int i, int deep, int t) {
  const int j = t - p.p0;
  if (j >= 0 && a.mask != nullptr) return (a.mask[(long long)(p.row + i) * a.words + (j >> 6)] >> (j & 63)) & 1;
  return j <= i && j > deep - a.window;
}
// the history's first position that a row sees, and the position behind the last key that it may see
__device__ __forceinline__ int first_key(const TreeArgs& a, const Portion& p, int deep) {
  const int t = max(p.p0 + deep - a.window + 1, 0);
  return a.mask != nullptr ? min(t, p.p0) : t;
}
__device__ __forceinline__ int end_key(const TreeArgs& a, const Portion& p, int i) { return a.mask != nullptr ? p.p0 + p.n : p.p0 + i + 1; }

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));            // (below 2^-126: 0; keeping those took three instructions more)
  return y;
}
__device__ __forceinline__ float lg2(float x) {
  float y;
  asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float y;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
  return y;
}
// two codes as fp16: e4m3 in the low 16 bits; int8 as the bytes code + 128, 0x64 each (1024 + 128 + code)
__device__ __forceinline__ uint32_t e4m3x2(uint32_t u) {
  const __half2_raw r = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)u, __NV_E4M3);
  return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t int8x2(uint32_t u) {
  const uint32_t off = 0x64806480u;                                // 1152
  const __half2 v = __hsub2(*reinterpret_cast<const __half2*>(&u), *reinterpret_cast<const __half2*>(&off));
  return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ uint32_t pack_f16x2(float lo, float hi) {
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
// The power of two that a row of queries is multiplied by on its way to fp16, and its inverse, by the bits (without sign) of its largest number: that becomes 2^14 to 2^15
struct Down {
  float by, back;
};
__device__ __forceinline__ Down down_of(uint32_t top) {
  const uint32_t e = min(max(top >> 7, 27u), 253u);
  return {__uint_as_float((268 - e) << 23), __uint_as_float((e - 14) << 23)};
}

// cap tanh(x / cap) = cap (1 - 2 / (1 + e^(2 x / cap))): off by up to 2^-21 of cap (the power 2^-22 of itself, the sum half a step, the quotient two), whatever x is, so that caps end where
// that is 2^-11, what weights of 11 bits are off by
constexpr float MOST_SOFTCAP = 1024.f;
__device__ __forceinline__ float capped(float x, float cap, float two_log2e_by_cap) { return cap - __fdividef(2.f * cap, 1.f + ex2(x * two_log2e_by_cap)); }

template <int KIND> __device__ __forceinline__ float cached(const uint8_t* head, int c) {
  if constexpr (KIND == LIA_CACHE_BF16) return __bfloat162float(reinterpret_cast<const bf16*>(head)[c]);
  else if constexpr (KIND == LIA_CACHE_INT8) return (float)reinterpret_cast<const int8_t*>(head)[c];
  else return __half2float(__half(__nv_cvt_fp8_to_halfraw(head[c], __NV_E4M3)));
}

// Row i, head h of a portion by one warp from the keys that it sees and no other, one after the other: for rows whose sums are not finite, where a number that the row does not see
// may have come in as 0 * inf.  y: channels lane, lane + 32, ...
// Some 1.3 us a key, so that one NaN or infinity among the values that a tile of rows reads costs far more than the call: a token behind 60000 positions 76 ms instead of 0.1, a chain of 8 behind
// 131003 160 ms, 64 tokens behind 2000 whose tile is one block's 60 ms (a warp's 32 rows one after the other).
template <int DIM, int VDIM, int KIND> __device__ __noinline__ void form_again(const TreeArgs& a, const Portion p, int i, int h, float* y) {
  constexpr int KN = DIM / 32, VN = VDIM / 32;
  const int lane = threadIdx.x & 31, g = h / a.rep, deep = depth_of(a, p, i);
  const float nan = __uint_as_float(0x7fc00000u), f = a.scale * (a.temp != nullptr ? a.temp[h] : 1.f);
  float q[KN], o[VN], m = -INFINITY, l = 0.f;
  for (int c = 0; c < KN; ++c) q[c] = __bfloat162float(a.q[(p.row + i) * a.ldq + h * DIM + c * 32 + lane]);
  for (int c = 0; c < VN; ++c) o[c] = 0.f;
  bool any = false;
  const int end = end_key(a, p, i);
  for (int t = first_key(a, p, deep); t < end; ++t) {
    if (!sees(a, p, i, deep, t)) continue;
    any = true;
    const uint8_t *kh = a.k.at(p.slot, t, g), *vh = a.v.at(p.slot, t, g);
    float s = 0.f;
    for (int c = 0; c < KN; ++c) s = fmaf(q[c], cached<KIND>(kh, c * 32 + lane), s);
    s = warp_sum(s) * f;
    if (KIND != LIA_CACHE_BF16) s *= a.k.scale_at(p.slot, g)[t];
    if (a.softcap > 0.f) s = a.softcap * tanhf(s / a.softcap);
    const float mn = fmaxf(m, s), keep = m == -INFINITY ? (mn == -INFINITY ? 1.f : 0.f) : expf(m - mn), w = s == -INFINITY ? 0.f : expf(s - mn);
    const float vs = KIND != LIA_CACHE_BF16 ? a.v.scale_at(p.slot, g)[t] : 1.f;
    l = l * keep + w;
    for (int c = 0; c < VN; ++c) o[c] = o[c] * keep + w * (cached<KIND>(vh, c * 32 + lane) * vs);
    m = mn;
  }
  for (int c = 0; c < VN; ++c) y[c] = !any ? 0.f : l > 0.f ? o[c] / l : nan;      // (all scores -inf, or NaN)
}

// A row's output from its sums (channels lane * N .. of a warp), or formed again
template <int DIM, int VDIM, int KIND> __device__ __forceinline__ void put_row(const TreeArgs& a, const Portion& p, int i, int h, const float* o, float l) {
  constexpr int N = VDIM / 32;
  const int lane = threadIdx.x & 31;
  const float inv = 1.f / l;
  float y[N], probe = 0.f;
#pragma unroll
  for (int c = 0; c < N; ++c) {
    y[c] = o[c] * inv;
    probe = fmaf(y[c], 0.f, probe);
  }
  bf16* dst = a.out + ((long long)(p.row + i) * a.H + h) * VDIM;
  if (__any_sync(0xffffffffu, !(probe == 0.f))) {                  // no key, or numbers that are not finite
    form_again<DIM, VDIM, KIND>(a, p, i, h, y);
#pragma unroll
    for (int c = 0; c < N; ++c) dst[c * 32 + lane] = __float2bfloat16_rn(y[c]);
    return;
  }
  if constexpr (N == 4) *reinterpret_cast<uint2*>(dst + lane * 4) = make_uint2(pack_bf16x2(y[0], y[1]), pack_bf16x2(y[2], y[3]));
  else *reinterpret_cast<uint32_t*>(dst + lane * 2) = pack_bf16x2(y[0], y[1]);
}

// The parts of a split history joined, always in the same order.  Warp per (row, head)
template <int DIM, int VDIM, int KIND> __global__ void __launch_bounds__(128) tree_attn_join_kernel(const __grid_constant__ TreeArgs a) {
  constexpr int N = VDIM / 32;
  pdl_launch_dependents();
  pdl_wait();
  const Portion p = portion_of(a, blockIdx.y);
  if (!p.held) {
    if (blockIdx.x == 0) nan_rows<VDIM>(a, p);
    return;
  }
  const int lane = threadIdx.x & 31, at = blockIdx.x * 4 + (threadIdx.x >> 5), i = at / a.H, h = at - i * a.H;
  if (i >= p.n) return;
  const long long rows = (long long)a.M * a.H, r = (long long)(p.row + i) * a.H + h;
  const float2* ml = reinterpret_cast<const float2*>(a.ws + a.splits * rows * VDIM) + r;
  float top = -INFINITY;
  for (int s = lane; s < a.splits; s += 32) top = fmaxf(top, ml[s * rows].x);
  top = warp_max(top);
  const float base = top == -INFINITY ? 0.f : top;
  float o[N] = {}, l = 0.f;
#pragma unroll 4
  for (int s = 0; s < a.splits; ++s) {
    const float2 x = ml[s * rows];
    const float f = ex2(x.x - base);
    const float* src = a.ws + (s * rows + r) * VDIM + lane * N;
    l = fmaf(x.y, f, l);
    float w[N];
    if constexpr (N == 4) *reinterpret_cast<float4*>(w) = *reinterpret_cast<const float4*>(src);
    else *reinterpret_cast<float2*>(w) = *reinterpret_cast<const float2*>(src);
#pragma unroll
    for (int c = 0; c < N; ++c) o[c] = fmaf(w[c], f, o[c]);
  }
  put_row<DIM, VDIM, KIND>(a, p, i, h, o, l);
}

}  // namespace
