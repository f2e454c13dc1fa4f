// Projections in 8-bit integers: out[m, n] = sx[m] sw[n] sum_k cx[m, k] cw[n, k], codes of 8 bits with a scale for each token and each channel, for sm_100a.
//
//   tokens   a = max |x[m]|, sx = a / 127, cx = rint(127 x / a)   (quantize_rows_kernel, a block a token; coder8.cuh)
//   sums     whole numbers of 32 bits, exact for up to 131071 products: whatever order they are added in, the bits are the same
//
// tcgen05.mma.kind::i8, both operands K-major from shared memory (TMA, 128-byte swizzle: 128 codes a row), sums in TMEM.  Two forms:
//   FEW    (up to 128 tokens; bound by the weights' bytes)  the weights' rows are the product's 128 rows, the tokens its 16 to 128 columns.  A CTA has a tile of 128 channels, or `parts` CTAs that are a
//          cluster share one along K and add up each other's sums by way of shared memory.  Two CTAs fit an SM, so that one's beginning and end lie under the other's loads, and memory shares itself out
//          among as many tiles as there are.  Weights are on their way while the tokens are quantised.
//   a token or two and matrices up to 64 Mi products, whose time is latency: int8_tokens_kernel, on the ordinary cores and in one launch.  Every block makes the tokens' codes for itself, in shared memory,
//          while its first weights are on their way; a warp has an equal part of the block's channels' codes.
//   MANY   (bound by the tensor cores, 86 % busy)  the tokens' rows are the product's rows: a CTA an SM on tiles of 128 x 256, or 128 or 64 where those would leave SMs idle.  (CTA pairs on 256 x 256 tiles,
//          cta_group::2, took 493 us where these took 622 in the same run, and came to a standstill once in some 20000 launches; why was not found, so they are not here.)
//
// us: 1 token of 2560 x 2560 5.1, latency; 64 tokens of 28672 x 7168 41, 5.0 TB/s of weights, 0.78 of the copy rate (both bf16, quantised on the way); 4096 tokens of it, of codes, 532 after a rest, 3160 TOP/s,
// and 620 to 635 at the 1305 to 1372 MHz that the power cap leaves after two seconds of it; bf16 tokens 580, and 662 at 1327 MHz.
// Quantisation: 28672 rows of 7168 bf16 numbers 114 us, 0.83 of the copy rate (issue slots 87 % busy); 4096 of them 17.7, of fp32 numbers 24.6 (0.91); 64 rows 2.5.
//
// Every wait is bounded; a CTA that gives one up makes its tile's outputs NaN and counts itself in lia_moe_timeouts_seen().
#include <cuda.h>

#include <mutex>

#include "coder8.cuh"
#include "common.cuh"
#include "umma.cuh"

int* lia_timeout_word();                                           // moe_sm100.cu

namespace {

constexpr int TILE = 128, KB = 128;                                // rows of a tile, codes (bytes) of a block of K
constexpr int MOST_K = 131071;                                     // 127 * 127 * K stays below 2^31 (and 128 * 128 * K)

// ------------------------------------------------------------------ tokens' codes
struct QuantArgs {
  const void* x;
  long long ldx, ldc;
  int8_t* codes;
  float* scale;
  int K, vec;
};
// Numbers 8 v .. 8 v + 7 of a row of K; those behind its end are zeros
template <typename T> __device__ __forceinline__ Raw8<T> load_of_row(const T* src, int v, int K, bool vec) {
  if (v * 8 >= K) return Raw8<T>{};
  if constexpr (sizeof(T) == 2) {                                  // rows of bf16 on 2-byte boundaries: by words of 4 bytes, of which only a row's first and last could lie outside it
    if (!vec && v > 0 && v * 8 + 8 < K) {
      const uintptr_t at = reinterpret_cast<uintptr_t>(src + v * 8);
      const uint32_t* p = reinterpret_cast<const uint32_t*>(at & ~(uintptr_t)3);
      uint32_t u[5];
#pragma unroll
      for (int i = 0; i < 4; ++i) u[i] = p[i];
      const bool half = at & 2;
      u[4] = half ? p[4] : 0u;
      Raw8<T> r;
      r.u[0] = half ? make_uint4(__byte_perm(u[0], u[1], 0x5432), __byte_perm(u[1], u[2], 0x5432), __byte_perm(u[2], u[3], 0x5432), __byte_perm(u[3], u[4], 0x5432)) : make_uint4(u[0], u[1], u[2], u[3]);
      return r;
    }
  }
  if (v * 8 + 8 <= K) return load8(src + v * 8, vec);
  T r[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) r[i] = v * 8 + i < K ? src[v * 8 + i] : (T)0.f;
  Raw8<T> u;
#pragma unroll
  for (int i = 0; i < (int)sizeof(T) / 2; ++i) u.u[i] = reinterpret_cast<const uint4*>(r)[i];
  return u;
}
constexpr int Q_HELD = 4;                                          // vectors of eight numbers that a thread holds: rows of 8192 numbers, or 32768, are read once

template <typename T, int Q_THREADS> __global__ void __launch_bounds__(Q_THREADS) quantize_rows_kernel(const __grid_constant__ QuantArgs a) {
  // In this order: the product behind asks for its weights before it waits, and may not begin before what came before this kernel (the weights' own quantisation, perhaps) has ended
  pdl_wait();
  pdl_launch_dependents();
  __shared__ uint32_t part[Q_THREADS / 32];
  const int t = threadIdx.x, vecs = (a.K + 7) / 8;
  const T* src = reinterpret_cast<const T*>(a.x) + (long long)blockIdx.x * a.ldx;
  auto load = [&](int v) { return load_of_row(src, v, a.K, a.vec); };
  Raw8<T> raw[Q_HELD];
#pragma unroll
  for (int i = 0; i < Q_HELD; ++i) raw[i] = load(t + i * Q_THREADS);
  uint32_t most = 0u;
#pragma unroll
  for (int i = 0; i < Q_HELD; ++i) most = most_of(raw[i], most);
  for (int v = t + Q_HELD * Q_THREADS; v < vecs; v += Q_THREADS) most = most_of(load(v), most);
  if constexpr (sizeof(T) == 2) most = max(most & 0xffffu, most >> 16) << 16;
  most = __reduce_max_sync(0xffffffffu, most);
  if ((t & 31) == 0) part[t >> 5] = most;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < Q_THREADS / 32; ++i) most = max(most, part[i]);
  const Coder<true> code(__uint_as_float(most));
  int8_t* dst = a.codes + (long long)blockIdx.x * a.ldc;
  auto put = [&](int v, const Raw8<T>& r) {
    if (v >= vecs) return;
    float f[8];
    numbers_of(r, f);
    const uint2 c = code(f);
    if (v * 8 + 8 <= a.K) {
      *reinterpret_cast<uint2*>(dst + v * 8) = c;
    } else {
      for (int i = v * 8; i < a.K; ++i) dst[i] = (int8_t)((i & 4 ? c.y : c.x) >> (8 * (i & 3)));
    }
  };
#pragma unroll
  for (int i = 0; i < Q_HELD; ++i) put(t + i * Q_THREADS, raw[i]);
  for (int v = t + Q_HELD * Q_THREADS; v < vecs; v += Q_THREADS) put(v, load(v));
  if (t == 0) a.scale[blockIdx.x] = code.scale;
}

// ------------------------------------------------------------------ a few tokens
struct TokenArgs {
  const void* x;
  const float* sx;                                                 // of codes that are given
  const int8_t* w;
  const float* sw;
  void* out;
  long long ldx, ldw;
  int N, K, vec, rows, steps;                                      // vec: vectors of 16 bytes may be read of x; channels of a block (an even number), blocks of 512 codes of a row
};
constexpr int T_WARPS = 16, T_THREADS = T_WARPS * 32, T_STEP = 512;                            // codes of a channel that a warp takes at once, 16 a lane
constexpr int T_ROWS = 1024, T_CODES = 32768;                       // most channels of a block; most numbers of the tokens
size_t token_smem(int M, int steps, int rows) { return (size_t)M * steps * T_STEP + (size_t)M * rows * 4; }
static_assert(T_CODES + 2 * T_STEP + 2 * T_ROWS * 4 <= 47 * 1024, "shared memory without asking for more");

template <typename T, int TOKENS, bool OUT32> __global__ void __launch_bounds__(T_THREADS, 1) int8_tokens_kernel(const __grid_constant__ TokenArgs a) {
  constexpr int UNITS = 4, HELD = T_CODES / 8 / T_THREADS / TOKENS;             // vectors of eight numbers that a thread has of each token
  extern __shared__ __align__(16) uint8_t smem_gen[];
  __shared__ uint32_t part[TOKENS][T_WARPS];
  __shared__ float sx_s[TOKENS];
  const int t = threadIdx.x, warp = t >> 5, lane = t & 31, width = a.steps * T_STEP;
  const int row0 = blockIdx.x * a.rows, rows = min(a.rows, a.N - row0);
  int* sums = reinterpret_cast<int*>(smem_gen + TOKENS * width);                               // [rows][TOKENS]
  // Units of two channels' 512 codes, the block's in a row: a sixteenth of them for each warp
  const int units = (rows + 1) / 2 * a.steps, first = (int)((long long)units * warp / T_WARPS), last = (int)((long long)units * (warp + 1) / T_WARPS);
  auto codes_at = [&](int pair, int k, int r) { return a.w + (long long)(row0 + 2 * pair + r) * a.ldw + k * T_STEP + lane * 16; };
  int pair = first / a.steps, k = first - pair * a.steps;          // of the units that are asked for next
  int ask = first;
  for (int u = ask, p = pair, s = k; u < min(last, ask + UNITS); ++u) {                        // to L2, where what comes before may still change them; the loads come behind the wait
#pragma unroll
    for (int r = 0; r < 2; ++r)
      if (lane % 2 == 0 && 2 * p + r < rows && s * T_STEP + lane * 16 < a.K) asm volatile("prefetch.global.L2 [%0];" ::"l"(codes_at(p, s, r)));
    if (++s == a.steps) s = 0, ++p;
  }
  pdl_wait();
  pdl_launch_dependents();
  uint4 w[UNITS][2], next[UNITS][2];
  auto ask_units = [&](uint4 (&to)[UNITS][2]) {
#pragma unroll
    for (int j = 0; j < UNITS; ++j) {
      const int left = a.K - k * T_STEP - lane * 16;               // of the row, from this lane's codes on
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        to[j][r] = make_uint4(0u, 0u, 0u, 0u);
        if (ask + j < last && 2 * pair + r < rows && left > 0) {
          const int8_t* src = codes_at(pair, k, r);
          if (left >= 16 || row0 + 2 * pair + r + 1 < a.N) {       // (what lies between two rows is multiplied by zeros)
            to[j][r] = __ldg(reinterpret_cast<const uint4*>(src));
          } else {
            uint32_t q[4] = {0u, 0u, 0u, 0u};
            for (int i = 0; i < left; ++i) q[i >> 2] |= (uint32_t)(uint8_t)src[i] << (8 * (i & 3));
            to[j][r] = make_uint4(q[0], q[1], q[2], q[3]);
          }
        }
      }
      if (++k == a.steps) k = 0, ++pair;
    }
    ask += UNITS;
  };
  int done = first, now = pair, at = k;                            // the unit that is multiplied next
  ask_units(w);

  // the tokens' codes, zeros behind their ends
  for (int i = t; i < a.rows * TOKENS; i += T_THREADS) sums[i] = 0;
  if constexpr (sizeof(T) == 1) {
    for (int i = t; i < TOKENS * (width / 16); i += T_THREADS) {
      const int m = i / (width / 16), c = (i - m * (width / 16)) * 16, left = a.K - c;
      uint4 q = make_uint4(0u, 0u, 0u, 0u);
      if (left > 0) {
        const int8_t* src = static_cast<const int8_t*>(a.x) + (long long)m * a.ldx + c;
        if (left >= 16) {
          q = ldg_act(reinterpret_cast<const bf16*>(src));
        } else {
          uint32_t b[4] = {0u, 0u, 0u, 0u};
          for (int e = 0; e < left; ++e) b[e >> 2] |= (uint32_t)(uint8_t)src[e] << (8 * (e & 3));
          q = make_uint4(b[0], b[1], b[2], b[3]);
        }
      }
      *reinterpret_cast<uint4*>(smem_gen + m * width + c) = q;
    }
    if (t < TOKENS) sx_s[t] = __ldcg(a.sx + t);
  } else {
    Raw8<T> raw[TOKENS][HELD];
#pragma unroll
    for (int m = 0; m < TOKENS; ++m)
#pragma unroll
      for (int i = 0; i < HELD; ++i) raw[m][i] = load_of_row(static_cast<const T*>(a.x) + m * a.ldx, t + i * T_THREADS, a.K, a.vec);
#pragma unroll
    for (int m = 0; m < TOKENS; ++m) {
      uint32_t most = 0u;
#pragma unroll
      for (int i = 0; i < HELD; ++i) most = most_of(raw[m][i], most);
      if constexpr (sizeof(T) == 2) most = max(most & 0xffffu, most >> 16) << 16;
      most = __reduce_max_sync(0xffffffffu, most);
      if (lane == 0) part[m][warp] = most;
    }
    __syncthreads();
#pragma unroll
    for (int m = 0; m < TOKENS; ++m) {
      const Coder<true> code(__uint_as_float(__reduce_max_sync(0xffffffffu, part[m][lane % T_WARPS])));
      auto put = [&](int v, const Raw8<T>& r) {
        if (v >= width / 8) return;
        float f[8];
        numbers_of(r, f);
        *reinterpret_cast<uint2*>(smem_gen + m * width + v * 8) = code(f);
      };
#pragma unroll
      for (int i = 0; i < HELD; ++i) put(t + i * T_THREADS, raw[m][i]);
      if (t == 0) sx_s[m] = code.scale;
    }
  }
  __syncthreads();

  int sum[TOKENS][2];
#pragma unroll
  for (int m = 0; m < TOKENS; ++m) sum[m][0] = sum[m][1] = 0;
  auto multiply = [&](const uint4 (&q)[UNITS][2]) {
#pragma unroll
    for (int j = 0; j < UNITS; ++j) {
      if (done >= last) return;
#pragma unroll
      for (int m = 0; m < TOKENS; ++m) {
        const int4 c = *reinterpret_cast<const int4*>(smem_gen + m * width + at * T_STEP + lane * 16);
#pragma unroll
        for (int r = 0; r < 2; ++r)
          sum[m][r] = __dp4a((int)q[j][r].w, c.w, __dp4a((int)q[j][r].z, c.z, __dp4a((int)q[j][r].y, c.y, __dp4a((int)q[j][r].x, c.x, sum[m][r]))));
      }
      ++done;
      ++at;
      if (at == a.steps || done == last) {                         // the channels' sums, or this warp's part of them
        int mine = 0;
#pragma unroll
        for (int m = 0; m < TOKENS; ++m)
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            const int s = __reduce_add_sync(0xffffffffu, sum[m][r]);
            if (lane == r * TOKENS + m) mine = s;
            sum[m][r] = 0;
          }
        if (lane < 2 * TOKENS) atomicAdd(sums + 2 * now * TOKENS + lane, mine);                // (whole numbers: in any order)
      }
      if (at == a.steps) at = 0, ++now;
    }
  };
  while (done < last) {
    ask_units(next);
    multiply(w);
#pragma unroll
    for (int j = 0; j < UNITS; ++j) w[j][0] = next[j][0], w[j][1] = next[j][1];
  }
  __syncthreads();
  for (int i = t; i < rows * TOKENS; i += T_THREADS) {
    const int m = i / rows, r = i - m * rows;
    const float y = (float)sums[r * TOKENS + m] * sx_s[m] * __ldg(a.sw + row0 + r);
    const size_t o = (size_t)m * a.N + row0 + r;
    if constexpr (OUT32) static_cast<float*>(a.out)[o] = y;
    else static_cast<bf16*>(a.out)[o] = __float2bfloat16_rn(y);
  }
}

// ------------------------------------------------------------------ products
struct Args {
  const float* sx;
  const float* sw;
  void* out;
  int* timeouts;
  int M, N, k_blocks, tiles_a, tiles_b, wide;                      // wide: rows of out are whole 16-byte vectors apart
  int parts;                                                       // FEW: CTAs that share a tile
};

// kind::i8: sums of 32-bit integers, both operands signed and K-major
__host__ __device__ constexpr uint32_t idesc_i8(int m, int n) { return (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24); }
__device__ __forceinline__ void mma_i8_if(uint32_t one, uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t@q tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(idesc),
               "r"(accumulate), "r"(one)
               : "memory");
}
template <bool FEW, int BN> struct Shape {
  static constexpr int A_BYTES = TILE * KB, B_BYTES = BN * KB, STAGE = A_BYTES + B_BYTES;
  static constexpr int OUT_WARPS = FEW ? 4 : 8, THREADS = 128 + 32 * OUT_WARPS;                // warps that take sums to outputs: two for 32 rows of a tile
  static constexpr int STAGING = FEW ? 0 : OUT_WARPS * 2048;       // 32 rows of 64 bytes for each of them
  static constexpr int STAGES = ((FEW ? 112640 : 228352) - STAGING) / STAGE > 8 ? 8 : ((FEW ? 112640 : 228352) - STAGING) / STAGE;    // (of FEW's, two blocks fit an SM)
  static constexpr int BARS = STAGES * STAGE + STAGING;
  static constexpr int SCALES = (BARS + (2 * STAGES + 5) * 8 + 8 + 15) / 16 * 16, SMEM = SCALES + (FEW ? BN : 2 * BN) * 4 + 1024;   // of the tokens, or of two tiles' channels
  static constexpr int COLS = FEW ? (BN < 32 ? 32 : BN) : 2 * BN;   // of TMEM: a tile's sums, or two tiles'
};

struct Work {
  int ta, tb, kb0, kb1;
};
// FEW: one tile, or part of one.  MANY: tile u = worker + i * workers, in groups of some rows of tiles, so that what runs at the same time shares operands in L2.
template <bool FEW> struct Sched {
  int k_blocks, tiles_a, tiles_b, group;
  unsigned pos, end, step;
  __device__ __forceinline__ explicit Sched(const Args& p) : k_blocks(p.k_blocks), tiles_a(p.tiles_a), tiles_b(p.tiles_b), group(16) {
    if (FEW) {
      const unsigned tile = blockIdx.x / (unsigned)p.parts, part = blockIdx.x - tile * (unsigned)p.parts;
      pos = tile * (unsigned)k_blocks + (unsigned)k_blocks * part / (unsigned)p.parts;         // (k_blocks is 1024 at most, and parts 8)
      end = tile * (unsigned)k_blocks + (unsigned)k_blocks * (part + 1) / (unsigned)p.parts;
      step = 0;
    } else {
      pos = blockIdx.x;
      step = gridDim.x;
      end = (unsigned)tiles_a * (unsigned)tiles_b;
    }
  }
  __device__ __forceinline__ bool next(Work& w) {
    if (pos >= end) return false;
    if (FEW) {
      w.ta = (int)(pos / (unsigned)k_blocks);
      w.tb = 0;
      w.kb0 = (int)(pos - (unsigned)w.ta * (unsigned)k_blocks);
      w.kb1 = min(k_blocks, w.kb0 + (int)(end - pos));
      pos += (unsigned)(w.kb1 - w.kb0);
    } else {
      const int u = (int)pos, size = group * tiles_b, first = u / size * group, gm = min(group, tiles_a - first), r = u % size;
      w.ta = first + r % gm;
      w.tb = r / gm;
      w.kb0 = 0;
      w.kb1 = k_blocks;
      pos += step;
    }
    return true;
  }
};

template <bool OUT32> __device__ __forceinline__ void put_one(void* out, size_t at, float y) {
  if constexpr (OUT32) reinterpret_cast<float*>(out)[at] = y;
  else reinterpret_cast<bf16*>(out)[at] = __float2bfloat16_rn(y);
}

template <bool FEW, int BN, bool OUT32>
__global__ void __launch_bounds__(Shape<FEW, BN>::THREADS, FEW ? 2 : 1) int8_gemm_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB, const __grid_constant__ Args p) {
  static_assert(FEW || BN >= 64, "two warps share the columns");
  using L = Shape<FEW, BN>;
  constexpr int STAGES = L::STAGES;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t smem = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* smem_gen = smem_raw + (smem - smem_u32(smem_raw));
  const uint32_t bars = smem + L::BARS;
  auto full = [&](int s) { return bars + 8u * s; };
  auto empty = [&](int s) { return bars + 8u * (STAGES + s); };
  auto tfull = [&](int a) { return bars + 8u * (2 * STAGES + a); };
  auto tempty = [&](int a) { return bars + 8u * (2 * STAGES + 2 + a); };
  const uint32_t drain = bars + 8u * (2 * STAGES + 4);
  volatile uint32_t* tmem_at = reinterpret_cast<volatile uint32_t*>(smem_gen + L::BARS + (2 * STAGES + 5) * 8);
  volatile int* dead = reinterpret_cast<volatile int*>(tmem_at + 1);
  const int warp = __shfl_sync(0xffffffffu, (int)threadIdx.x >> 5, 0), lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(&tmA) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&tmB) : "memory");
    *dead = 0;
  }
  if (warp == 1 && lane == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(full(s), 1);
      mbar_init(empty(s), 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(tfull(a), 1);
      mbar_init(tempty(a), L::OUT_WARPS);
    }
    mbar_init(drain, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 2) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32((const void*)tmem_at)), "r"((uint32_t)L::COLS) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tcgen05_fence_before();
  __syncthreads();
  tcgen05_fence_after();
  const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_at, 0);
  pdl_launch_dependents();                                         // (only weights are touched before pdl_wait)
  int issued = 0;                                                  // blocks that the loading lane has asked for

  if (warp == 0) {
    // ================================================================ loads
    if (lane == 0) {
      int early = 0;
      if (FEW) {                                                   // weights, which no kernel writes, before the tokens' codes are there
        Sched<FEW> s(p);
        Work w;
        while (early < STAGES && s.next(w))
          for (int kb = w.kb0; kb < w.kb1 && early < STAGES; ++kb, ++early) {
            mbar_expect_tx(full(early), L::STAGE);
            tma_load_block(smem + early * L::STAGE, &tmA, kb, w.ta * TILE, full(early));
          }
      }
      pdl_wait();
      Sched<FEW> s(p);
      Work w;
      int stage = 0;
      uint32_t phase = 0;
      bool alive = true;
      while (alive && s.next(w))
        for (int kb = w.kb0; kb < w.kb1; ++kb) {
          const uint32_t sa = smem + stage * L::STAGE, sb = sa + L::A_BYTES;
          if (FEW && issued < early) {
            tma_load_block(sb, &tmB, kb, 0, full(stage));
          } else {
            if (!(alive = wait_for(empty(stage), phase ^ 1u, dead))) break;
            mbar_expect_tx(full(stage), L::STAGE);
            tma_load_block(sa, &tmA, kb, w.ta * TILE, full(stage));
            tma_load_block(sb, &tmB, kb, w.tb * BN, full(stage));
          }
          ++issued;
          if (++stage == STAGES) {
            stage = 0;
            phase ^= 1u;
          }
        }
    }
  } else if (warp == 1) {
    // ================================================================ products
    const uint32_t one = elect_one();
    constexpr uint32_t idesc = idesc_i8(TILE, BN);
    Sched<FEW> s(p);
    Work w;
    int stage = 0, acc = 0;
    uint32_t phase = 0, acc_phase = 0;
    bool alive = true;
    while (alive && s.next(w)) {
      if (!(alive = warp_wait(tempty(acc), acc_phase ^ 1u, dead))) break;
      tcgen05_fence_after();
      const uint32_t d = tmem + (uint32_t)(acc * BN);
      for (int kb = w.kb0; kb < w.kb1; ++kb) {
        if (!(alive = warp_wait(full(stage), phase, dead))) break;
        tcgen05_fence_after();
        const uint32_t sa = smem + stage * L::STAGE;
        const uint64_t da = make_smem_desc(sa), db = make_smem_desc(sa + L::A_BYTES);
#pragma unroll
        for (int k = 0; k < KB / 32; ++k) {                      // 32 codes on are 32 bytes inside the swizzled row: + 2 in the address field
          mma_i8_if(one, d, da + (uint64_t)(2 * k), db + (uint64_t)(2 * k), idesc, (kb > w.kb0 || k > 0) ? 1u : 0u);
        }
        commit_if(one, empty(stage));
        if (++stage == STAGES) {
          stage = 0;
          phase ^= 1u;
        }
      }
      if (!alive) break;
      commit_if(one, tfull(acc));
      acc ^= 1;
      if (acc == 0) acc_phase ^= 1u;
    }
  } else if (warp >= 4) {
    // ================================================================ sums to outputs
    const int ew = warp & 3, half = (warp - 4) >> 2;               // TMEM lanes 32 ew .. 32 ew + 31; of MANY's two warps for them each has every other 32 columns
    auto out_warps_meet = [] { asm volatile("bar.sync 1, %0;" ::"n"(L::OUT_WARPS * 32) : "memory"); };
    pdl_wait();
    float* scales_s = reinterpret_cast<float*>(smem_gen + L::SCALES);                          // (read one by one between the outputs' stores they cost an L2 round trip each: 128 tokens 30 us)
    if (FEW) {
      const int i = ew * 32 + lane;
      if (i < BN) scales_s[i] = i < p.M ? __ldcg(p.sx + i) : 0.f;
      out_warps_meet();
    }
    Sched<FEW> s(p);
    Work w;
    int acc = 0;
    uint32_t acc_phase = 0;
    bool alive = true;
    while (s.next(w)) {
      if (!FEW) {                                                  // the channels' scales, while the sums are on their way; zeros behind the last (the buffer before the last tile's has been read)
        for (int i = threadIdx.x - 128; i < BN; i += L::OUT_WARPS * 32) scales_s[acc * BN + i] = w.tb * BN + i < p.N ? __ldg(p.sw + w.tb * BN + i) : 0.f;
        out_warps_meet();
      }
      alive = __all_sync(0xffffffffu, alive && wait_for(tfull(acc), acc_phase, dead));
      tcgen05_fence_after();
      const uint32_t taddr = tmem + (uint32_t)(acc * BN) + ((uint32_t)(ew * 32) << 16);
      auto give_back = [&] {                                       // the sums are read
        tcgen05_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(tempty(acc));
      };
      if constexpr (FEW) {
        // a lane has one channel, its columns are the tokens: to shared memory where the operands were, [tokens][TILE]
        int* sums = reinterpret_cast<int*>(smem_gen) + ew * 32 + lane;
        constexpr int CH = BN < 32 ? BN : 32;
        if (alive) {
#pragma unroll 1
          for (int c = 0; c < BN && c < p.M; c += CH) {
            uint32_t v[CH];
            if constexpr (CH == 32) tmem_ld32(taddr + c, v);
            else tmem_ld16(taddr + c, v);
            tmem_ld_wait();
#pragma unroll
            for (int j = 0; j < CH; ++j)
              if (c + j < p.M) sums[(c + j) * TILE] = (int)v[j];
          }
        }
      } else {
        // a lane has one token, its columns are channels: through shared memory to whole rows
        const int row0 = w.ta * TILE + ew * 32, m = row0 + lane;
        const float sx = m < p.M ? __ldcg(p.sx + m) : 0.f;
        const uint32_t stg = smem + STAGES * L::STAGE + (warp - 4) * 2048;
        constexpr int PER = OUT32 ? 4 : 8, COLS = OUT32 ? 16 : 32; // columns of 16 bytes; of 64, which 32 rows of are in shared memory at a time
#pragma unroll 1
        for (int c0 = 32 * half; c0 < BN; c0 += 64) {
          uint32_t v[32];
          if (alive) {
            tmem_ld32(taddr + c0, v);
            tmem_ld_wait();
            if (c0 + 64 >= BN) give_back();                        // (by now they are in registers)
          }
          const float4* sw = reinterpret_cast<const float4*>(scales_s + acc * BN + c0);
#pragma unroll
          for (int j = 0; j < 32; j += 4) {
            const float4 w4 = sw[j / 4];
            const float f[4] = {w4.x, w4.y, w4.z, w4.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) v[j + e] = __float_as_uint(alive ? (float)(int)v[j + e] * sx * f[e] : NAN);
          }
#pragma unroll
          for (int part = 0; part < 32 / COLS; ++part) {
#pragma unroll
            for (int chunk = 0; chunk < 4; ++chunk) {              // each pair of rows' chunks turned by the pair, so that neither side of the transposition collides
              const uint32_t* u = v + part * COLS + chunk * PER;
              uint4 q;
              if constexpr (OUT32) q = make_uint4(u[0], u[1], u[2], u[3]);
              else q = pack8(reinterpret_cast<const float*>(u));
              asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(stg + lane * 64 + ((chunk ^ (lane >> 1 & 3)) << 4)), "r"(q.x), "r"(q.y), "r"(q.z), "r"(q.w) : "memory");
            }
            __syncwarp();
            const int n0 = w.tb * BN + c0 + part * COLS;
            if (p.wide) {
#pragma unroll
              for (int it = 0; it < 4; ++it) {
                const int r = it * 8 + (lane >> 2), chunk = lane & 3, n = n0 + chunk * PER;
                uint4 q;
                asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(q.x), "=r"(q.y), "=r"(q.z), "=r"(q.w) : "r"(stg + r * 64 + ((chunk ^ (r >> 1 & 3)) << 4)));
                if (row0 + r < p.M && n < p.N) *reinterpret_cast<uint4*>(reinterpret_cast<uint8_t*>(p.out) + ((size_t)(row0 + r) * p.N + n) * (OUT32 ? 4 : 2)) = q;
              }
            } else {                                               // rows that begin anywhere: neighbouring lanes, neighbouring numbers (202 x 26373 outputs by fours and eights a lane: 33 us)
              constexpr int AT_ONCE = 32 / COLS;                   // rows
              const int e = lane % COLS, rows = min(32, p.M - row0);
              const bool in = n0 + e < p.N;
#pragma unroll 8
              for (int r0 = 0; r0 < 32; r0 += AT_ONCE) {
                const int r = r0 + lane / COLS;
                const uint32_t from = stg + r * 64 + (((e / PER) ^ (r >> 1 & 3)) << 4) + e % PER * (16 / PER);
                const size_t at = (size_t)(row0 + r) * p.N + n0 + e;
                if constexpr (OUT32) {
                  uint32_t x;
                  asm volatile("ld.shared.b32 %0, [%1];" : "=r"(x) : "r"(from));
                  if (in && r < rows) reinterpret_cast<uint32_t*>(p.out)[at] = x;
                } else {
                  uint16_t x;
                  asm volatile("ld.shared.b16 %0, [%1];" : "=h"(x) : "r"(from));
                  if (in && r < rows) reinterpret_cast<uint16_t*>(p.out)[at] = x;
                }
              }
            }
            __syncwarp();
          }
        }
      }
      acc ^= 1;
      if (acc == 0) acc_phase ^= 1u;
    }
  }

  tcgen05_fence_before();
  __syncthreads();
  if (FEW) {
    // ================================================================ a cluster's parts of a tile: each CTA adds up and writes some of the outputs, four channels a thread at a time
    pdl_wait();
    if (p.parts > 1) cluster_barrier();
    const int rank4 = (int)(blockIdx.x % (unsigned)p.parts), first = (p.M * (TILE / 4) * rank4 / p.parts), last = (p.M * (TILE / 4) * (rank4 + 1) / p.parts), n0 = (int)(blockIdx.x / (unsigned)p.parts) * TILE;
    const float* sx_s = reinterpret_cast<const float*>(smem_gen + L::SCALES);
    bool bad = false;
    for (int o = 0; o < p.parts; ++o) bad |= cluster_ld_u32(cluster_place(const_cast<const int*>(dead), o)) != 0u;
    if (p.wide) {
      for (int i = first + (int)threadIdx.x; i < last; i += 256) {
        const int m = i / (TILE / 4), n = n0 + i % (TILE / 4) * 4;
        int4 sum = make_int4(0, 0, 0, 0);
#pragma unroll 4
        for (int o = 0; o < p.parts; ++o) {
          const float4 f = cluster_ld_f4(cluster_place(smem_gen + (size_t)i * 16, o));
          sum.x += __float_as_int(f.x), sum.y += __float_as_int(f.y), sum.z += __float_as_int(f.z), sum.w += __float_as_int(f.w);
        }
        if (n >= p.N) continue;                                    // (whole vectors, as rows are)
        const int v[4] = {sum.x, sum.y, sum.z, sum.w};
        float y[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) y[j] = bad ? NAN : (float)v[j] * sx_s[m] * __ldg(p.sw + n + j);
        const size_t at = (size_t)m * p.N + n;
        if constexpr (OUT32) *reinterpret_cast<float4*>(reinterpret_cast<float*>(p.out) + at) = make_float4(y[0], y[1], y[2], y[3]);
        else *reinterpret_cast<uint2*>(reinterpret_cast<bf16*>(p.out) + at) = make_uint2(pack_bf16x2(y[0], y[1]), pack_bf16x2(y[2], y[3]));
      }
    } else {                                                       // rows that begin anywhere: one channel a thread
      for (int i = first * 4 + (int)threadIdx.x; i < last * 4; i += 256) {
        const int m = i / TILE, n = n0 + i % TILE;
        int sum = 0;
#pragma unroll 4
        for (int o = 0; o < p.parts; ++o) sum += (int)cluster_ld_u32(cluster_place(smem_gen + (size_t)i * 4, o));
        if (n < p.N) put_one<OUT32>(p.out, (size_t)m * p.N + n, bad ? NAN : (float)sum * sx_s[m] * __ldg(p.sw + n));
      }
    }
    __syncwarp();                                                  // (lanes leave these loops after different rounds, and TMEM is given back by a whole warp)
  }
  if (*dead) {                                                     // loads and products in flight end before shared memory and TMEM are given back
    if (threadIdx.x == 0) {
      atomicAdd_system(p.timeouts, 1);
      for (int i = 0; i < STAGES && i < issued; ++i) {
        const int n = issued - 1 - i;
        wait_in_flight(full(n % STAGES), (uint32_t)(n / STAGES) & 1u);
      }
    }
    if (warp == 1) {
      const uint32_t one = elect_one();
      commit_if(one, drain);
      wait_in_flight(drain, 0u);
    }
    __syncthreads();
  }
  if (FEW && p.parts > 1) cluster_barrier();                       // nobody leaves while others may read its sums
  if (warp == 2) {
    tcgen05_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"((uint32_t)L::COLS) : "memory");
  }
}

// ------------------------------------------------------------------ host
// codes [rows, K], `ld` bytes from row to row: boxes of 128 codes x box_rows, what lies outside reads as zeros
int make_tmap(CUtensorMap* map, const void* base, int rows, int K, long long ld, int box_rows) {
  PFN_encodeTiled enc = get_encode();
  LIA_CHECK_ARG(enc, "cuTensorMapEncodeTiled entry point not available (no CUDA driver?)");
  cuuint64_t dims[2] = {(cuuint64_t)K, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)ld};
  cuuint32_t box[2] = {(cuuint32_t)KB, (cuuint32_t)box_rows}, one[2] = {1, 1};
  const CUresult r = enc(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                         CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) {
    lia_set_error("cuTensorMapEncodeTiled failed with CUresult %d (rows=%d K=%d ld=%lld)", (int)r, rows, K, ld);
    return LIA_ERR_CUDA;
  }
  return LIA_OK;
}

struct Plan {
  bool few;
  int bn, grid, tiles_a, tiles_b, k_blocks, parts;                 // parts: CTAs of a cluster that share a tile
};
Plan plan_of(int M, int N, int K) {
  Plan p{};
  const int sms = lia_sm_count();
  p.k_blocks = (K + KB - 1) / KB;
  p.few = M <= 128;
  if (p.few) {
    p.bn = M <= 16 ? 16 : M <= 32 ? 32 : M <= 64 ? 64 : 128;
    p.tiles_a = (N + TILE - 1) / TILE;
    p.tiles_b = 1;
    // Sharing a tile costs a cluster's meeting, 1 to 2 us, and pays as long as the CTAs fit two an SM; eight of them only where the tiles are few and long.  us with 1 | 2 | 4 | 8 parts, 64 tokens:
    // 1024 x 1024 9.0 | 8.2 | 7.4 | 7.2; 2560 x 2560 12.1 | 10.2 | 8.8 | 9.6; 1024 x 8192 22.5 | 15.6 | 11.5 | 10.7; 7168 x 7168 24.2 | 19.1 | 17.0 | 23.6; 12288 x 4096 19.3 | 18.0 | 21.4;
    // 28672 x 7168 41.4 | 46.5.  (As spans of equal length over one CTA an SM, whose shared tiles met by way of global memory, 2560 x 2560 took 18, 28672 x 7168 49.)
    p.parts = 1;
    if (p.k_blocks >= 40 && p.tiles_a * 8 <= sms * 11 / 10) p.parts = 8;
    else if (p.k_blocks >= 4 && p.tiles_a * 4 <= sms * 8 / 5) p.parts = 4;
    else if (p.k_blocks >= 4 && p.tiles_a * 2 <= sms * 8 / 5) p.parts = 2;
    p.grid = p.tiles_a * p.parts;
    return p;
  }
  auto tiles = [&](int cols) { return (long long)((M + TILE - 1) / TILE) * ((N + cols - 1) / cols); };
  long long least = -1;
  auto offer = [&](int bn, long long time) {
    if (least >= 0 && time >= least) return;
    least = time;
    p.bn = bn;
  };
  // ns: a call's own, and for each round what its blocks of K take or, behind the first one, what its sums take on their way out if that is longer; fitted to 90 shapes.  us by tiles 256 wide | 128 | 64,
  // of codes: 256 tokens of 1024 x 1024 7.4 | 5.5 | 4.9, of 7168 x 7168 21 | 15 | 24; 1000 tokens of it 40 | 46 | 76; 1150 of 23176 x 416 24 | 28 | 37; 4096 of 28672 x 7168 532 | 633 | 1022 after a rest,
  // 627 at 1340 MHz | 737 at 1425 | 1158 at 1690 under the power cap.
  auto ns = [&](long long n, long long once, int block, int sums) {
    const long long products = (long long)p.k_blocks * block;
    return once + products + ((n + sms - 1) / sms - 1) * (products > sums ? products : sums);
  };
  offer(256, ns(tiles(256), 6000, 533, 3300));
  offer(128, ns(tiles(128), 5000, 342, 2150));
  offer(64, ns(tiles(64), 4550, 253, 1600));
  p.tiles_a = (M + TILE - 1) / TILE;
  p.tiles_b = (N + p.bn - 1) / p.bn;
  const long long units = (long long)p.tiles_a * p.tiles_b;
  p.grid = (int)(units < sms ? units : sms);
  return p;
}
// of a workspace: codes and scales of the tokens, unless they are given
struct Rooms {
  size_t scales, bytes;
  long long ldc;
};
Rooms rooms_of(int M, int K, bool given) {
  Rooms r{};
  r.ldc = ((long long)K + 15) / 16 * 16;
  if (given) return r;
  r.scales = ((size_t)M * r.ldc + 255) / 256 * 256;
  r.bytes = r.scales + (size_t)M * sizeof(float);
  return r;
}

template <bool FEW, int BN, bool OUT32> int launch(const Plan& pl, const CUtensorMap& tmA, const CUtensorMap& tmB, const Args& a, bool early, cudaStream_t stream) {
  using L = Shape<FEW, BN>;
  static_assert(L::SMEM <= (FEW ? 115712 : 232448) && L::STAGES >= 3 && (!FEW || L::STAGES * L::STAGE >= BN * TILE * 4), "shared memory");
  auto kernel = int8_gemm_kernel<FEW, BN, OUT32>;
  static bool configured[64] = {};                                 // per device
  int dev = 0;
  LIA_CUDA(cudaGetDevice(&dev));
  if (dev >= 64 || !configured[dev]) {
    LIA_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, L::SMEM));
    if (dev < 64) configured[dev] = true;
  }
  if (pl.parts > 1) LIA_CUDA(lia_launch_cluster_as(early, pl.parts, kernel, dim3(pl.grid), dim3(L::THREADS), L::SMEM, stream, tmA, tmB, a));
  else LIA_CUDA(lia_launch_as(early, kernel, dim3(pl.grid), dim3(L::THREADS), L::SMEM, stream, tmA, tmB, a));
  return LIA_OK;
}
template <bool OUT32> int launch_plan(const Plan& pl, const CUtensorMap& tmA, const CUtensorMap& tmB, const Args& a, bool early, cudaStream_t stream) {
  if (pl.few) {
    switch (pl.bn) {
      case 16: return launch<true, 16, OUT32>(pl, tmA, tmB, a, early, stream);
      case 32: return launch<true, 32, OUT32>(pl, tmA, tmB, a, early, stream);
      case 64: return launch<true, 64, OUT32>(pl, tmA, tmB, a, early, stream);
      default: return launch<true, 128, OUT32>(pl, tmA, tmB, a, early, stream);
    }
  }
  switch (pl.bn) {
    case 256: return launch<false, 256, OUT32>(pl, tmA, tmB, a, early, stream);
    case 128: return launch<false, 128, OUT32>(pl, tmA, tmB, a, early, stream);
    default: return launch<false, 64, OUT32>(pl, tmA, tmB, a, early, stream);
  }
}

int quantize(const void* x, int act_f32, long long ldx, int8_t* codes, long long ldc, float* scale, int M, int K, cudaStream_t stream) {
  const QuantArgs q{x, ldx, ldc, codes, scale, K, reinterpret_cast<uintptr_t>(x) % 16 == 0 && ldx % (act_f32 ? 4 : 8) == 0};
  // a block of 256 threads holds a row of 8192 numbers, one of 1024 four times that; longer rows are read twice
  if (K > 8 * Q_HELD * 256) {
    if (act_f32) LIA_CUDA(lia_launch(quantize_rows_kernel<float, 1024>, dim3(M), dim3(1024), 0, stream, q));
    else LIA_CUDA(lia_launch(quantize_rows_kernel<bf16, 1024>, dim3(M), dim3(1024), 0, stream, q));
  } else {
    if (act_f32) LIA_CUDA(lia_launch(quantize_rows_kernel<float, 256>, dim3(M), dim3(256), 0, stream, q));
    else LIA_CUDA(lia_launch(quantize_rows_kernel<bf16, 256>, dim3(M), dim3(256), 0, stream, q));
  }
  return LIA_OK;
}

// us with quantisation and tcgen05 | in one launch, bf16 tokens: 1 of 1024 x 1024 5.9 | 4.8, of 2560 x 2560 7.5 | 5.3, of 1000 x 8192 8.4 | 5.8, of 64 x 28672 12.5 | 6.2, of 7168 x 7168 14.0 | 13.3, of
// 50272 x 2560 26.0 | 25.7, of 28672 x 7168 35.6 | 37.3, of 200000 x 64 21 | 26 (and in two rounds, 200000 x 256, 23 | 26); 2 of 2560 x 2560 7.5 | 5.7, of 1000 x 8192 8.4 | 6.8, of 2048 x 28672 16.7 | 20.1 (every block quantises the tokens);
// 4, by a form of it that is not here, of 2560 x 2560 7.5 | 7.0, of 1000 x 8192 8.5 | 8.5, of 7168 x 7168 14.0 | 16.3.  A call is shorter by a launch and an allocation too.
bool few_tokens(int M, int N, int K) { return M <= 2 && K >= T_STEP / 2 && (long long)M * K <= T_CODES && (long long)M * N * K <= 1ll << 26 && N <= lia_sm_count() * T_ROWS; }

template <typename T, bool OUT32> int launch_tokens(TokenArgs a, int M, cudaStream_t stream) {
  const int sms = lia_sm_count();                                  // as many channels for each
  a.rows = ((a.N + sms - 1) / sms + 1) / 2 * 2;
  LIA_CUDA(lia_launch(M == 1 ? int8_tokens_kernel<T, 1, OUT32> : int8_tokens_kernel<T, 2, OUT32>, dim3((a.N + a.rows - 1) / a.rows), dim3(T_THREADS), token_smem(M, a.steps, a.rows), stream, a));
  return LIA_OK;
}
template <bool OUT32> int launch_tokens(int x_type, const TokenArgs& a, int M, cudaStream_t stream) {
  switch (x_type) {
    case LIA_X_BF16: return launch_tokens<bf16, OUT32>(a, M, stream);
    case LIA_X_F32: return launch_tokens<float, OUT32>(a, M, stream);
    default: return launch_tokens<int8_t, OUT32>(a, M, stream);
  }
}

}  // namespace

extern "C" int lia_quantize_rows(const void* x, int act_f32, long long ldx, void* codes, long long ldc, float* scale, int M, int K, lia_stream_t stream) {
  LIA_CHECK_ARG(M >= 0 && K > 0 && ldx >= K && ldc >= K, "lia_quantize_rows: bad sizes");
  if (M == 0) return LIA_OK;
  LIA_CHECK_ARG(x && codes && scale, "lia_quantize_rows: null pointer");
  LIA_CHECK_ARG(reinterpret_cast<uintptr_t>(codes) % 8 == 0 && ldc % 8 == 0, "lia_quantize_rows: rows of codes have to be whole 8-byte vectors apart");
  return quantize(x, act_f32, ldx, static_cast<int8_t*>(codes), ldc, scale, M, K, reinterpret_cast<cudaStream_t>(stream));
}

extern "C" size_t lia_linear_int8_workspace_bytes(int x_type, int M, int N, int K) {
  if (M <= 0 || N <= 0 || K <= 0 || K > MOST_K) return 0;
  return rooms_of(M, K, x_type == LIA_X_INT8 || few_tokens(M, N, K)).bytes;
}

extern "C" int lia_linear_int8(const void* x, int x_type, long long ldx, const float* x_scale, const void* w, long long ldw, const float* w_scale, void* out, int out_f32, int M, int N, int K,
                               void* ws, size_t ws_bytes, lia_stream_t stream_) {
  cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_);
  const bool given = x_type == LIA_X_INT8;
  LIA_CHECK_ARG(x_type >= LIA_X_BF16 && x_type <= LIA_X_INT8, "lia_linear_int8: unknown type %d of tokens", x_type);
  LIA_CHECK_ARG(M >= 0 && N > 0 && K > 0 && ldx >= K && ldw >= K, "lia_linear_int8: bad sizes");
  LIA_CHECK_ARG(K <= MOST_K, "lia_linear_int8: sums of %d products do not fit 32 bits (at most %d)", K, MOST_K);
  if (M == 0) return LIA_OK;
  LIA_CHECK_ARG(x && w && w_scale && out && (given == (x_scale != nullptr)), "lia_linear_int8: null pointer, or scales of tokens that are not codes");
  LIA_CHECK_ARG(reinterpret_cast<uintptr_t>(w) % 16 == 0 && ldw % 16 == 0 && (!given || (reinterpret_cast<uintptr_t>(x) % 16 == 0 && ldx % 16 == 0)),
                "lia_linear_int8: rows of codes have to be whole 16-byte vectors apart");
  if (few_tokens(M, N, K)) {
    const int vec = given || (reinterpret_cast<uintptr_t>(x) % 16 == 0 && ldx % (x_type == LIA_X_F32 ? 4 : 8) == 0);
    const TokenArgs a{x, x_scale, static_cast<const int8_t*>(w), w_scale, out, ldx, ldw, N, K, vec, 0, (K + T_STEP - 1) / T_STEP};
    return out_f32 ? launch_tokens<true>(x_type, a, M, stream) : launch_tokens<false>(x_type, a, M, stream);
  }
  const Plan pl = plan_of(M, N, K);
  LIA_CHECK_ARG((long long)pl.tiles_a * pl.k_blocks < (1ll << 31) && (long long)pl.tiles_a * pl.tiles_b < (1ll << 31), "lia_linear_int8: too large (M=%d N=%d K=%d)", M, N, K);
  const Rooms r = rooms_of(M, K, given);
  LIA_CHECK_ARG(r.bytes == 0 || (ws && ws_bytes >= r.bytes && reinterpret_cast<uintptr_t>(ws) % 16 == 0), "lia_linear_int8: needs a workspace of %zu bytes", r.bytes);
  uint8_t* base = static_cast<uint8_t*>(ws);
  const void* codes = given ? x : base;
  const long long ldc = given ? ldx : r.ldc;
  CUtensorMap tmX, tmW;
  int rc = make_tmap(&tmX, codes, M, K, ldc, pl.few ? pl.bn : TILE);
  if (rc == LIA_OK) rc = make_tmap(&tmW, w, N, K, ldw, pl.few ? TILE : pl.bn);
  if (rc != LIA_OK) return rc;
  Args a{given ? x_scale : reinterpret_cast<float*>(base + r.scales), w_scale, out, lia_timeout_word(), M, N, pl.k_blocks,
         pl.tiles_a, pl.tiles_b, reinterpret_cast<uintptr_t>(out) % 16 == 0 && (long long)N * (out_f32 ? 4 : 2) % 16 == 0, pl.parts};
  LIA_CHECK_ARG(a.timeouts, "lia_linear_int8: no memory for the count of waits that ran out");
  if (!given) rc = quantize(x, x_type == LIA_X_F32, ldx, reinterpret_cast<int8_t*>(base), r.ldc, reinterpret_cast<float*>(base + r.scales), M, K, stream);
  if (rc != LIA_OK) return rc;
  const bool early = !given;                                       // (right behind another kernel, which may have written the weights, the product does not begin before that has ended)
  return pl.few ? (out_f32 ? launch_plan<true>(pl, tmW, tmX, a, early, stream) : launch_plan<false>(pl, tmW, tmX, a, early, stream))
                : (out_f32 ? launch_plan<true>(pl, tmX, tmW, a, early, stream) : launch_plan<false>(pl, tmX, tmW, a, early, stream));
}
