// Log probabilities of given tokens, the entropy of the distribution and the most likely tokens, from a model's logits.
//
//   with m = max x, L = sum e^(x - m), A = sum e^(x - m) (x - m):   log p(t) = x_t - m - ln L,   entropy = ln L - A / L
//
// One pass over the logits: every thread keeps a running maximum with its L and A (a larger maximum multiplies both by a power and moves A by L times the step), and every warp the 32
// largest logits that it has met, sorted, one a lane, as whole numbers that order by value and then by lower id.  A logit that is not above the `top`-th of them costs one comparison (and
// most blocks of 512 one vote); the others are gathered in shared memory, 32 at a time sorted across the warp's lanes and merged with the list.  The first block would have the list take
// all of its logits; instead the top-th largest of its lanes' maxima is a bound that at most some dozens reach.
// Few rows share out a row's blocks over several blocks of threads, and a second kernel joins the parts (in the same order each time).
//
// Memory bounds it for many rows (a logit is read once, eight instructions each), the latency of one block of logits and two launches for few.
#include "common.cuh"

namespace {

constexpr int WARPS = 8, THREADS = WARPS * 32, MAX_TOP = 32;
constexpr float LOG2E = 1.4426950408889634f;
typedef unsigned long long u64;

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
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
__device__ __forceinline__ void raise_to(Sums& s, float m) {
  if (s.m != -INFINITY) {
    const float d = s.m - m, f = ex2(d * LOG2E);
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
__device__ __forceinline__ float logit_of(u64 k) {
  const uint32_t o = (uint32_t)(k >> 32);
  return __uint_as_float(o & 0x80000000u ? o & 0x7fffffffu : ~o);
}

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
  Sums* part_sums;                                                 // [M][splits], then
  u64* part_lists;                                                 // [M][splits][32]
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

template <typename T>
__global__ void __launch_bounds__(THREADS, 4) token_logprobs_kernel(const Args a) {
  constexpr int N = Vec<T>::N, U = Vec<T>::U, SHARE = N * U;
  __shared__ u64 gathered[WARPS][64];
  __shared__ Sums warp_sums[WARPS];
  pdl_launch_dependents();
  pdl_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, row = blockIdx.x / a.splits, split = blockIdx.x - row * a.splits;
  const T* x = reinterpret_cast<const T*>(a.logits) + row * a.ld;
  const int skew = (int)(reinterpret_cast<uintptr_t>(x) % 16 / sizeof(T));            // the row begins inside a 16-byte vector
  const uint4* vecs = reinterpret_cast<const uint4*>(x - skew);
  const int nv = (a.V + skew + N - 1) / N, blocks = (nv + 32 * U - 1) / (32 * U);
  const int b0 = (int)((long long)blocks * split / a.splits), b1 = (int)((long long)blocks * (split + 1) / a.splits);

  auto load = [&](int b, uint4* u) {
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const int v = b * 32 * U + i * 32 + lane, e = v * N - skew;
      if (b < b1 && v < nv) {
        if (e >= 0 && e + N <= a.V) {
          u[i] = ldg_act(vecs + v);
        } else {                                                   // the row's ends: what is not its own counts as -inf
          T t[N];
#pragma unroll
          for (int j = 0; j < N; ++j) t[j] = e + j >= 0 && e + j < a.V ? x[e + j] : (T)(-INFINITY);
          u[i] = *reinterpret_cast<const uint4*>(t);
        }
      } else {
        const T low = (T)(-INFINITY);
        T t[N];
#pragma unroll
        for (int j = 0; j < N; ++j) t[j] = low;
        u[i] = *reinterpret_cast<const uint4*>(t);
      }
    }
  };

  Sums s{-INFINITY, 0.f, 0.f};
  u64 list = 0;
  int held = 0;                                                    // gathered logits
  float bound = __uint_as_float(0x7fc00000u);                      // the top-th of the list; NaN: it has not that many
  u64* mine = gathered[warp];
  auto take = [&](int n) {                                         // the first n <= 32 gathered ones join the list
    __syncwarp();
    list = merge_down(list, sort_up(lane < n ? mine[lane] : 0, lane), lane);
    const u64 rest = lane + 32 < held ? mine[lane + 32] : 0;
    __syncwarp();
    mine[lane] = rest;
    held -= n;
    const u64 last = __shfl_sync(0xffffffffu, list, a.top - 1);
    bound = last ? logit_of(last) : __uint_as_float(0x7fc00000u);
    __syncwarp();
  };

  uint4 u[U], next[U];
  bool first = true;
  load(b0 + warp, u);
  for (int b = b0 + warp; b < b1; b += WARPS) {
    load(b + WARPS, next);
    float f[SHARE], m = -INFINITY;
#pragma unroll
    for (int i = 0; i < U; ++i) Vec<T>::unpack(u[i], f + i * N);
#pragma unroll
    for (int i = 0; i < SHARE; ++i) m = fmaxf(m, f[i]);
    if (m > s.m) raise_to(s, m);
    const float base = s.m == -INFINITY ? 0.f : s.m;
    float L[2] = {0.f, 0.f}, A[2] = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < SHARE; ++i) {
      const float y = max_nan(f[i] - base, -200.f), e = ex2(y * LOG2E);                 // (e^-200 is 0; -inf would make 0 * inf of A)
      L[i & 1] += e;
      A[i & 1] = fmaf(e, y, A[i & 1]);
    }
    s.L += L[0] + L[1];
    s.A += A[0] + A[1];
    if (a.top > 0) {
      float least = bound;
      bool equal = false;                                          // the first block's bound is not in the list yet
      if (first) {
        const u64 best = sort_up(key_of(m, 0), lane);              // (rising: the top-th largest is top from the end)
        least = logit_of(__shfl_sync(0xffffffffu, best, 32 - a.top));
        equal = true;
        first = false;
      }
      if (__any_sync(0xffffffffu, equal || !(m <= least))) {
#pragma unroll
        for (int i = 0; i < SHARE; ++i) {
          const int id = (b * 32 * U + (i / N) * 32 + lane) * N - skew + i % N;
          const bool in = (equal ? !(f[i] < least) : !(f[i] <= least)) && id >= 0 && id < a.V;
          const unsigned who = __ballot_sync(0xffffffffu, in);
          if (who) {
            if (in) mine[held + __popc(who & ((1u << lane) - 1u))] = key_of(f[i], id);
            held += __popc(who);
            if (held >= 32) {
              take(32);
              if (!equal) least = bound;
            }
          }
        }
      }
    }
#pragma unroll
    for (int i = 0; i < U; ++i) u[i] = next[i];
  }
  if (a.top > 0 && held > 0) take(held);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) join(s, from_lane(s, o));
  __syncwarp();
  if (a.top > 0) mine[31 - lane] = list;                           // rising
  if (lane == 0) warp_sums[warp] = s;
  __syncthreads();
  if (warp != 0) return;
  s = warp_sums[0];
  for (int w = 1; w < WARPS; ++w) {
    join(s, warp_sums[w]);
    if (a.top > 0) list = merge_down(list, gathered[w][lane], lane);
  }
  if (a.splits == 1) {
    finish<T>(a, row, s, list, lane);
  } else {
    if (lane == 0) a.part_sums[blockIdx.x] = s;
    if (a.top > 0) a.part_lists[(long long)blockIdx.x * 32 + lane] = list;
  }
}

template <typename T>
__global__ void __launch_bounds__(32) token_logprobs_join_kernel(const Args a) {
  pdl_launch_dependents();
  pdl_wait();
  const int row = blockIdx.x, lane = threadIdx.x;
  const long long at = (long long)row * a.splits;
  Sums s = a.part_sums[at];
  u64 list = a.top > 0 ? a.part_lists[at * 32 + lane] : 0;
  for (int i = 1; i < a.splits; ++i) {
    join(s, a.part_sums[at + i]);
    if (a.top > 0) list = merge_down(list, a.part_lists[(at + i) * 32 + 31 - lane], lane);
  }
  finish<T>(a, row, s, list, lane);
}

// Blocks of threads of a row: as many as fill the GPU four blocks an SM, none with less than one block of logits a warp
int splits_of(int M, int V, int act_f32) {
  const int per = WARPS * 512, most = (V + per - 1) / per, want = (4 * lia_sm_count() + M - 1) / M;
  (void)act_f32;
  return want < 1 ? 1 : want < most ? want : most;
}
size_t floats_of(int M, int splits) { return splits > 1 ? (size_t)M * splits * (4 + 64) : 0; }

}  // namespace

extern "C" size_t lia_token_logprobs_workspace_floats(int M, int V, int act_f32) { return M > 0 && V > 0 ? floats_of(M, splits_of(M, V, act_f32)) : 0; }

extern "C" int lia_token_logprobs(const void* logits, int act_f32, long long ld, int M, int V, const int64_t* tokens, int n, float* logp, float* entropy, int top, float* top_logp,
                                  int64_t* top_ids, float* ws, size_t ws_floats, lia_stream_t stream_) {
  cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_);
  LIA_CHECK_ARG(M >= 0 && V > 0 && V < (1 << 30) && ld >= V && top >= 0 && top <= MAX_TOP && top <= V && n >= 0, "lia_token_logprobs: bad sizes (top is at most %d and V)", MAX_TOP);
  if (M == 0) return LIA_OK;
  LIA_CHECK_ARG(logits && entropy && (n == 0 || (tokens && logp)) && (top == 0 || (top_logp && top_ids)), "lia_token_logprobs: null pointer");
  LIA_CHECK_ARG(reinterpret_cast<uintptr_t>(logits) % (act_f32 ? 4 : 2) == 0, "lia_token_logprobs: misaligned logits");
  const int splits = splits_of(M, V, act_f32);
  LIA_CHECK_ARG(splits == 1 || (ws && ws_floats >= floats_of(M, splits) && reinterpret_cast<uintptr_t>(ws) % 16 == 0), "lia_token_logprobs: needs a workspace of %zu floats", floats_of(M, splits));
  LIA_CHECK_ARG((long long)M * splits < (1ll << 31), "lia_token_logprobs: too many rows");
  Args a{logits, ld, M, V, splits, top, n, reinterpret_cast<const long long*>(tokens), logp, entropy, top_logp, reinterpret_cast<long long*>(top_ids), reinterpret_cast<Sums*>(ws),
         reinterpret_cast<u64*>(ws + (size_t)M * splits * 4)};
  if (act_f32) LIA_CUDA(lia_launch(token_logprobs_kernel<float>, dim3(M * splits), dim3(THREADS), 0, stream, a));
  else LIA_CUDA(lia_launch(token_logprobs_kernel<bf16>, dim3(M * splits), dim3(THREADS), 0, stream, a));
  if (splits > 1) {
    if (act_f32) LIA_CUDA(lia_launch(token_logprobs_join_kernel<float>, dim3(M), dim3(32), 0, stream, a));
    else LIA_CUDA(lia_launch(token_logprobs_join_kernel<bf16>, dim3(M), dim3(32), 0, stream, a));
  }
  return LIA_OK;
}
