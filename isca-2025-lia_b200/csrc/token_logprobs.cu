// Log probabilities of given tokens, the entropy of the distribution and the most likely tokens, from a model's logits.
//
//   with m = max x, L = sum e^(x - m), A = sum e^(x - m) (x - m):   log p(t) = x_t - m - ln L,   entropy = ln L - A / L
//
// One pass over the logits: every thread keeps a running maximum with its L and A (a larger maximum multiplies both by a power and moves A by L times the step).  The largest ones are
// found from what that leaves: the top-th largest of the 256 threads' maxima is reached by at least `top` logits and, as the largest ones seldom share a thread, by few more; every thread
// knows the maxima of four parts of its logits, so that only the parts that reach it are read again (a fortieth of the row, from L2), by all lanes of their warps.  What reaches the bound is sorted across a warp's lanes,
// as whole numbers that order by value and then by lower id.  (With lists of the largest ones kept by every warp through the pass 4096 rows took 577 us instead of 172.)
// Few rows share out a row over a cluster of up to eight blocks of threads, whose first one joins the parts (in the same order each time).
//
// Bound, at 4096 rows of 50272 logits: fp32 by memory, 131 us without the largest ones (96 % of the rate of a copy) and 156 with the 20 largest; bf16, half the bytes, by instructions:
// 96 and 150 us.  (Issued are some 17 a logit, counted with fp32 and the 20 largest, issue slots 61 % busy.)  Few rows by the latency of one block of logits and of sorting: four rows 9 us.
#include "pairs.cuh"

namespace {

constexpr int WARPS = 8, THREADS = WARPS * 32, MAX_TOP = 32;
constexpr float LOG2E = 1.4426950408889634f;
typedef unsigned long long u64;

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));            // (below 2^-126 of the largest: 0)
  return y;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float y;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
  return y;
}

// A row's sums: m the largest logit, L = sum e^(x - m), A = sum e^(x - m) (x - m)
struct alignas(16) Sums {
  float m, L, A;
};
// (a step counts as 200 at most, where its power is 0 already: of sums whose maximum is a mask of the type's least number, d or d * L would be infinite, and 0 times that NaN)
__device__ __forceinline__ void raise_to(Sums& s, float m) {
  if (s.m != -INFINITY) {
    const float d = fmaxf(s.m - m, -200.f), f = ex2(d * LOG2E);
    s.A = f * fmaf(d, s.L, s.A);
    s.L *= f;
  }
  s.m = m;
}
__device__ __forceinline__ void join(Sums& a, Sums b) {
  if (b.m > a.m) raise_to(a, b.m);
  else if (a.m != b.m) raise_to(b, a.m);
  a.L += b.L;
  a.A += b.A;
}
__device__ __forceinline__ Sums from_lane(const Sums& s, int o) {
  return {__shfl_xor_sync(0xffffffffu, s.m, o), __shfl_xor_sync(0xffffffffu, s.L, o), __shfl_xor_sync(0xffffffffu, s.A, o)};
}

// Logit and id as one whole number: larger for a larger logit, of equal ones for the lower id; NaN as -inf.  0: none.
__device__ __forceinline__ u64 key_of(float x, int id) {
  x = x != x ? -INFINITY : x == 0.f ? 0.f : x;                     // (-0 and 0 are equal)
  const uint32_t b = __float_as_uint(x), o = b & 0x80000000u ? ~b : b | 0x80000000u;
  return (u64)o << 32 | (uint32_t)~id;
}
__device__ __forceinline__ int id_of(u64 k) { return ~(int)(uint32_t)k; }
// neighbours o lanes apart put the larger one first where `first_larger`
__device__ __forceinline__ u64 exchange(u64 v, int o, bool keep_larger) {
  const u64 w = __shfl_xor_sync(0xffffffffu, v, o);
  return (v > w) == keep_larger ? v : w;
}
__device__ __forceinline__ u64 sort_up(u64 v, int lane) {
#pragma unroll
  for (int k = 2; k <= 32; k <<= 1)
#pragma unroll
    for (int o = k >> 1; o > 0; o >>= 1) v = exchange(v, o, ((lane & k) == 0) == ((lane & o) != 0));
  return v;
}
// list falls with the lane, more rises: the 32 largest of both, falling
__device__ __forceinline__ u64 merge_down(u64 list, u64 more, int lane) {
  u64 v = list > more ? list : more;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = exchange(v, o, (lane & o) == 0);
  return v;
}

// the same of plain whole numbers, for bounds
__device__ __forceinline__ uint32_t sort_down32(uint32_t v, int lane) {
#pragma unroll
  for (int k = 2; k <= 32; k <<= 1)
#pragma unroll
    for (int o = k >> 1; o > 0; o >>= 1) {
      const uint32_t w = __shfl_xor_sync(0xffffffffu, v, o);
      v = ((lane & k) == 0) == ((lane & o) == 0) ? max(v, w) : min(v, w);
    }
  return v;
}
__device__ __forceinline__ uint32_t merge_down32(uint32_t list, uint32_t more, int lane) {
  uint32_t v = max(list, more);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const uint32_t w = __shfl_xor_sync(0xffffffffu, v, o);
    v = (lane & o) == 0 ? max(v, w) : min(v, w);
  }
  return v;
}
template <typename T> struct Vec;
template <> struct Vec<float> {
  static constexpr int N = 4, U = 4;                               // logits of a vector; vectors of a lane's share of a block
  static __device__ __forceinline__ void unpack(const uint4& u, float* f) {
    f[0] = __uint_as_float(u.x); f[1] = __uint_as_float(u.y); f[2] = __uint_as_float(u.z); f[3] = __uint_as_float(u.w);
  }
};
template <> struct Vec<bf16> {
  static constexpr int N = 8, U = 2;
  static __device__ __forceinline__ void unpack(const uint4& u, float* f) { unpack8(u, f); }
};

struct Args {
  const void* logits;
  long long ld;
  int M, V, splits, top, n;
  const long long* tokens;
  float *logp, *entropy, *top_logp;
  long long* top_ids;
};

__device__ __forceinline__ float logit(const float* p) { return *p; }
__device__ __forceinline__ float logit(const bf16* p) { return __bfloat162float(*p); }

// A row's results by one warp that has its sums and its list
template <typename T> __device__ __forceinline__ void finish(const Args& a, int row, const Sums& s, u64 list, int lane) {
  const float lnL = logf(s.L);                                     // (NaN where the row holds NaN or +inf; m is -inf where it holds no more than that)
  for (int j = lane; j < a.n; j += 32) {
    const long long t = a.tokens[(long long)row * a.n + j];
    a.logp[(long long)row * a.n + j] = t >= 0 && t < a.V ? logit(reinterpret_cast<const T*>(a.logits) + row * a.ld + t) - s.m - lnL : __uint_as_float(0x7fc00000u);
  }
  if (lane == 0) a.entropy[row] = s.m == -INFINITY ? __uint_as_float(0x7fc00000u) : lnL - s.A / s.L;
  if (lane < a.top) {
    a.top_ids[(long long)row * a.top + lane] = id_of(list);
    const float x = logit(reinterpret_cast<const T*>(a.logits) + row * a.ld + id_of(list));
    a.top_logp[(long long)row * a.top + lane] = x - s.m - lnL;
  }
}

// The lists of a block's W warps (each in lists[warp], falling; a power of two of them) become one, in warp 0's hands
template <int W> __device__ __forceinline__ u64 join_lists(u64 list, u64 (*lists)[32], int warp, int lane) {
#pragma unroll
  for (int half = W / 2; half > 0; half >>= 1) {
    if (warp >= half && warp < 2 * half) lists[warp][31 - lane] = list;                 // rising
    __syncthreads();
    if (warp < half) list = merge_down(list, lists[warp + half][lane], lane);
  }
  return list;
}

template <typename T>
__global__ void __launch_bounds__(THREADS, 4) token_logprobs_kernel(const Args a) {
  constexpr int N = Vec<T>::N, U = Vec<T>::U, SHARE = N * U, ROOM = 1024, PARTS = 4;
  __shared__ u64 found[ROOM];                                      // the logits that reach the bound
  __shared__ u64 lists[WARPS][32];
  __shared__ int count;
  __shared__ uint32_t bound;
  __shared__ uint8_t hot[WARPS][32 * PARTS];
  __shared__ uint32_t bounds[WARPS][32];
  __shared__ Sums warp_sums[WARPS];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, row = blockIdx.x / a.splits, split = blockIdx.x - row * a.splits;
  pdl_launch_dependents();
  pdl_wait();
  const T* x = reinterpret_cast<const T*>(a.logits) + row * a.ld;
  const int skew = (int)(reinterpret_cast<uintptr_t>(x) % 16 / sizeof(T));            // the row begins inside a 16-byte vector
  const uint4* vecs = reinterpret_cast<const uint4*>(x - skew);
  const int nv = (a.V + skew + N - 1) / N, blocks = (nv + 32 * U - 1) / (32 * U);
  const int b0 = (int)((long long)blocks * split / a.splits), b1 = (int)((long long)blocks * (split + 1) / a.splits);

  auto vector = [&](int v) {                                       // what is not the row's own counts as -inf
    const int e = v * N - skew;
    if (v < nv && e >= 0 && e + N <= a.V) return ldg_act(vecs + v);
    T t[N];
#pragma unroll
    for (int j = 0; j < N; ++j) t[j] = e + j >= 0 && e + j < a.V ? x[e + j] : (T)(-INFINITY);
    return *reinterpret_cast<const uint4*>(t);
  };
  auto load = [&](int b, uint4* u) {
    if (b < b1 && (b > 0 || skew == 0) && (b + 1) * 32 * SHARE - skew <= a.V) {
#pragma unroll
      for (int i = 0; i < U; ++i) u[i] = ldg_act(vecs + b * 32 * U + i * 32 + lane);
    } else {
#pragma unroll
      for (int i = 0; i < U; ++i) u[i] = vector((b < b1 ? b * 32 * U : nv) + i * 32 + lane);
    }
  };

  // ---- sums, and every thread's maximum
  Sums s{-INFINITY, 0.f, 0.f};
  float parts[PARTS];                                              // the maximum of every fourth of the thread's shares
#pragma unroll
  for (int q = 0; q < PARTS; ++q) parts[q] = -INFINITY;
  uint4 u[U], next[U];
  load(b0 + warp, u);
  for (int b = b0 + warp, turn = 0; b < b1; b += WARPS, turn = (turn + 1) & (PARTS - 1)) {
    load(b + WARPS, next);
    float f[SHARE], m = -INFINITY;
#pragma unroll
    for (int i = 0; i < U; ++i) Vec<T>::unpack(u[i], f + i * N);
#pragma unroll
    for (int i = 0; i < SHARE; ++i) m = fmaxf(m, f[i]);
    if (m > s.m) raise_to(s, m);
#pragma unroll
    for (int q = 0; q < PARTS; ++q) parts[q] = turn == q ? fmaxf(parts[q], m) : parts[q];
    const float base = s.m == -INFINITY ? 0.f : s.m;
    f32x2 L = 0ull, A = 0ull;
#pragma unroll
    for (int i = 0; i < SHARE; i += 2) {
      float y0, y1;
      unpack2(add2(pack2(f[i], f[i + 1]), both(-base)), y0, y1);
      const f32x2 y = pack2(max_nan(y0, -200.f), max_nan(y1, -200.f));                  // (e^-200 is 0; -inf would make 0 * inf of A)
      unpack2(mul2(y, both(LOG2E)), y0, y1);
      const f32x2 e = pack2(ex2(y0), ex2(y1));
      L = add2(L, e);
      A = fma2(e, y, A);
    }
    float p0, p1;
    unpack2(L, p0, p1);
    s.L += p0 + p1;
    unpack2(A, p0, p1);
    s.A += p0 + p1;
#pragma unroll
    for (int i = 0; i < U; ++i) u[i] = next[i];
  }

  u64 list = 0;
  if (a.top > 0) {
    // ---- the top-th largest of the threads' maxima bounds what can be among the top
    if (threadIdx.x == 0) count = 0;
    uint32_t best = sort_down32((uint32_t)(key_of(s.m, 0) >> 32), lane);
#pragma unroll
    for (int half = WARPS / 2; half > 0; half >>= 1) {
      if (warp >= half && warp < 2 * half) bounds[warp][31 - lane] = best;                // rising
      __syncthreads();
      if (warp < half) best = merge_down32(best, bounds[warp + half][lane], lane);
    }
    if (threadIdx.x == a.top - 1) bound = best;
    __syncthreads();
    // ---- the shares that hold something that reaches it, once more by all lanes of their warp
    int shares = 0;
#pragma unroll
    for (int q = 0; q < PARTS; ++q) {
      const bool in = (uint32_t)(key_of(parts[q], 0) >> 32) >= bound;
      const unsigned who = __ballot_sync(0xffffffffu, in);
      if (in) hot[warp][shares + __popc(who & ((1u << lane) - 1u))] = (uint8_t)(lane + 32 * q);
      shares += __popc(who);
    }
    __syncwarp();
    const int turns = b0 + warp < b1 ? (b1 - b0 - warp + WARPS - 1) / WARPS : 0, each = (turns + PARTS - 1) / PARTS * U, items = shares * each;
    for (int t0 = lane; t0 < items; t0 += 128) {
      uint4 w[4];
      int v[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int t = t0 + j * 32, h = t / each, r = t - h * each, from = t < items ? hot[warp][h] : 0, turn = r / U * PARTS + (from >> 5);
        v[j] = t < items && turn < turns ? (b0 + warp + turn * WARPS) * 32 * U + r % U * 32 + (from & 31) : nv;
        w[j] = vector(v[j]);
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        float f[N];
        Vec<T>::unpack(w[j], f);
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const u64 k = key_of(f[i], v[j] * N - skew + i);
          if ((uint32_t)(k >> 32) >= bound && id_of(k) >= 0 && id_of(k) < a.V && v[j] < nv) {
            const int at = atomicAdd(&count, 1);                   // (in any order: they are sorted)
            if (at < ROOM) found[at] = k;
          }
        }
      }
    }
    __syncthreads();
    const int n = count;
    if (n <= ROOM) {                                               // some more than top, 32 by 32 by warp 0
      list = 0;
      if (warp == 0)
        for (int i = 0; i < n; i += 32) list = merge_down(list, sort_up(i + lane < n ? found[i + lane] : 0, lane), lane);
    } else {                                                       // many equal ones: every warp looks at all of its logits again, with the least of its list for a bound
      list = 0;
      u64 least = 0;
      for (int b = b0 + warp; b < b1; b += WARPS)
        for (int i = 0; i < U; ++i) {
          float f[N];
          const int v = b * 32 * U + i * 32 + lane;
          Vec<T>::unpack(vector(v), f);
          for (int j = 0; j < N; ++j) {
            const int id = v * N - skew + j;
            const u64 k = id >= 0 && id < a.V ? key_of(f[j], id) : 0;
            if (__any_sync(0xffffffffu, k > least)) {
              list = merge_down(list, sort_up(k, lane), lane);
              least = __shfl_sync(0xffffffffu, list, 31);
            }
          }
        }
      list = join_lists<WARPS>(list, lists, warp, lane);
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) join(s, from_lane(s, o));
  if (lane == 0) warp_sums[warp] = s;
  __syncthreads();
  if (warp == 0) {
    s = warp_sums[0];
    for (int w = 1; w < WARPS; ++w) join(s, warp_sums[w]);
  }
  if (a.splits > 1) {                                              // the row's other blocks are the cluster's: the first one fetches their parts, a warp each
    __syncthreads();                                               // (the sums and lists of the warps have been read)
    if (warp == 0) {
      if (lane == 0) warp_sums[0] = s;
      lists[0][lane] = list;
    }
    cluster_barrier();
    if (split == 0) {
      list = 0;
      s = {-INFINITY, 0.f, 0.f};
      if (warp < a.splits) {
        const float4 q = cluster_ld_f4(cluster_place(&warp_sums[0], warp));
        s = {q.x, q.y, q.z};
        if (a.top > 0) list = cluster_ld64(cluster_place(&lists[0][lane], warp));
      }
      __syncthreads();                                             // (its own part among them)
      if (lane == 0) warp_sums[warp] = s;
      if (a.top > 0) list = join_lists<WARPS>(list, lists, warp, lane);
      __syncthreads();
      if (warp == 0) {
        s = warp_sums[0];
        for (int w = 1; w < a.splits; ++w) join(s, warp_sums[w]);
      }
    }
  }
  if (warp == 0 && split == 0) finish<T>(a, row, s, list, lane);
  if (a.splits > 1) cluster_barrier();                             // (no block leaves while it is read)
}

// Blocks of threads of a row, one cluster of them: 1, 2, 4 or 8, as many as fill the GPU four blocks an SM, none with less than a block of logits a warp
int splits_of(int M, int V) {
  int s = WARPS;
  while (s > 1 && ((long long)s * M > 4 * lia_sm_count() || s * WARPS * 512 > V + WARPS * 512)) s /= 2;
  return s;
}

}  // namespace

extern "C" int lia_token_logprobs(const void* logits, int act_f32, long long ld, int M, int V, const int64_t* tokens, int n, float* logp, float* entropy, int top, float* top_logp,
                                  int64_t* top_ids, lia_stream_t stream_) {
  cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_);
  LIA_CHECK_ARG(M >= 0 && V > 0 && V < (1 << 30) && ld >= V && top >= 0 && top <= MAX_TOP && top <= V && n >= 0, "lia_token_logprobs: bad sizes (top is at most %d and V)", MAX_TOP);
  if (M == 0) return LIA_OK;
  LIA_CHECK_ARG(logits && entropy && (n == 0 || (tokens && logp)) && (top == 0 || (top_logp && top_ids)), "lia_token_logprobs: null pointer");
  LIA_CHECK_ARG(reinterpret_cast<uintptr_t>(logits) % (act_f32 ? 4 : 2) == 0, "lia_token_logprobs: misaligned logits");
  const int splits = splits_of(M, V);
  const Args a{logits, ld, M, V, splits, top, n, reinterpret_cast<const long long*>(tokens), logp, entropy, top_logp, reinterpret_cast<long long*>(top_ids)};
  auto go = [&](auto kernel) {
    return splits == 1 ? lia_launch(kernel, dim3(M), dim3(THREADS), 0, stream, a) : lia_launch_cluster(splits, kernel, dim3(M * splits), dim3(THREADS), 0, stream, a);
  };
  LIA_CUDA(act_f32 ? go(token_logprobs_kernel<float>) : go(token_logprobs_kernel<bf16>));
  return LIA_OK;
}
