// Attention of drafted tokens (tree_attn.cu has the formulas) for many rows of a key head, on tcgen05: 128 rows of (token, head) to a block, or 256 where there are more.
//
//   warps 0-3, 4-7   two groups, each with a maximum, a sum and weighted values of its own; a thread has one row, which is one lane of TMEM.  Of 256 rows each group has 128; of up
//                    to 128 both have the same rows and take the history's blocks of 64 keys in turn, and they meet at the end.
//   warps 8-15       bring keys and values: 16 bytes a lane from memory, 8-bit codes as fp16, into shared memory as the products want them (128-byte swizzle).  Positions behind the last key
//                    become zeros, so that nothing unwritten is multiplied.
//   warp 16          the products (three more are there for their registers)
// TMEM, 512 columns: group s has the scores of two blocks, one being worked on and the next one, at 128 s and 128 s + 64, in their place its weights (fp16, or two bf16 parts), and its
// weighted values at 256 + 128 s.  (With one block's scores and the queries in TMEM too, a group waited for scores that are issued behind its weights' products; the queries in shared memory
// cost nothing: 6 KB a product are less than shared memory gives in that time.)
// The weighted values stay in TMEM from block to block.  Weights are relative to a maximum that moves only when a row has exceeded it by 2^8 (they fit fp16 up to there); only then
// its group multiplies what it has, behind the products of its last block.
//
// 8-bit scales: a key's is multiplied into its scores in fp32.  A value's is multiplied into its channels on their way to fp16, relative to the power of two REF of the first keys' largest
// (rounded to 11 bits twice: 2^-11 each, as the weights are), which leaves the softmax one instruction less in three.  A value whose scale is not within 2^-8 to 2^6 of REF, one of nothing or NaN
// among them, stays as it is and its scale joins the exponent (tree_attn.cu); a block with one takes a slower way.
//
// What bounds it: at 128 rows and more the softmax -- a row of 64 scores is one thread's chain of loads from TMEM, a maximum, powers, sums and stores, and two groups of four warps hide little of
// one another's (with the products halved the time stays as it is, and sixteen warps of it had too few registers) -- at 2.7 times the 512 clocks that 64 x 128 powers take; with fewer rows
// memory (700 clocks for 64 keys of 8 bits, 1400 of bf16).  A call behind a single position takes 16 us with 256 rows a block, 10 with up to 128: programs are loaded, and what depends on the portion, one
// behind the other.  A tree of 64 tokens behind 131003 positions, 32 heads on 8: int8 212 us, bf16 205; its products would take 83 at the tensor cores' rate, its bytes 42 and 82.
// Keys' scales are held 16 at a time (32: 240 us, for registers).
// The issuing warp's block numbers are made uniform by a shuffle: without, each product took twice its instructions.
#include "pairs.cuh"
#include "tree_attn.cuh"
#include "umma.cuh"

int* lia_formed_again_word();                                      // moe_sm100.cu

namespace {

constexpr int ROWS = 128, KEYS = 64, THREADS = 640, LOADERS = 256, ISSUER = 16;
constexpr int SOFTMAX_REGS = 128, LOADER_REGS = 96, OTHER_REGS = 32; // of a thread, by what its four warps do (setmaxnreg: multiples of 8); the launch gives 96
constexpr int LAUNCH_REGS = 96;
static_assert(SOFTMAX_REGS >= LAUNCH_REGS && LOADER_REGS <= LAUNCH_REGS && OTHER_REGS <= LAUNCH_REGS && 2 * SOFTMAX_REGS + 2 * LOADER_REGS + OTHER_REGS <= THREADS / 128 * LAUNCH_REGS, "shares");
constexpr uint32_t VALUES = 256;
constexpr float SLACK = 8.f;                                       // how far, in powers of two, weights may exceed 1

template <int DIM, int VDIM, int KIND, bool PAIR>
struct Tc {
  static constexpr bool BITS8 = KIND != LIA_CACHE_BF16;
  static constexpr int SLAB = KEYS * 128;                          // 64 channels of 16 bits of a block's keys
  static constexpr int K_BYTES = DIM / 64 * SLAB, V_BYTES = VDIM / 64 * SLAB, STAGE = K_BYTES + V_BYTES;
  static constexpr int Q_SLAB = ROWS * 128, Q_BYTES = DIM / 64 * Q_SLAB;                        // a group's queries
  static constexpr int ALL_Q = (PAIR ? 2 : 1) * Q_BYTES, ROOM = (221184 - ALL_Q) / STAGE, STAGES = ROOM > 8 ? 8 : ROOM;
  static constexpr int KT = DIM * (BITS8 ? 1 : 2) / 16, VT = VDIM * (BITS8 ? 1 : 2) / 16;      // lanes of a key, of a value
  static constexpr int KN = KEYS * KT / LOADERS, VN = KEYS * VT / LOADERS;                       // vectors of a lane
  static constexpr int AHEAD = BITS8 ? 2 : 1;                      // blocks of 16 or 32 KB on their way from memory (more: more instructions to bring, 5 to 30 % slower with four)
  static constexpr float LIFT = BITS8 ? 7.f : 0.f;                 // weights are 2^(x - maximum + LIFT): below 2^15 in fp16
};
struct Tail {
  float ks[8][KEYS], lv[8][KEYS], rv[8][KEYS];                     // of a stage's keys: scale; of its values: log2 of what is left of the scale, and the inverse of that
  uint64_t odd[8];                                                 // of a stage: a byte for every warp that has brought a value with a scale far from REF
  float2 ml[ROWS];
  float row_f[2 * ROWS];                                           // what a row's products with keys are multiplied by
  uint64_t full[8], empty[8], s_full[2][2], p_full[2][2], o_done[2], q_full, drain;
  uint32_t tmem;
  int dead;
};

// where a lane's 16 channels of an 8-bit head lie among the products' columns: of 128, the first eight in one slab and the others in the next (so that the lanes that write them together
// write to different banks), of 64 side by side
template <int DIM> __device__ __forceinline__ int place_of(int j, int half) { return DIM == 128 ? half * 64 + j * 8 : j * 16 + half * 8; }

template <int KIND> __device__ __forceinline__ void widen(const uint4& u, uint4& lo, uint4& hi) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
  uint32_t r[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (KIND == LIA_CACHE_INT8) {
      const uint32_t x = w[i] ^ 0x80808080u;
      r[2 * i] = int8x2(__byte_perm(x, 0x64646464u, 0x4140));
      r[2 * i + 1] = int8x2(__byte_perm(x, 0x64646464u, 0x4342));
    } else {
      r[2 * i] = e4m3x2(w[i] & 0xffffu);
      r[2 * i + 1] = e4m3x2(w[i] >> 16);
    }
  }
  lo = make_uint4(r[0], r[1], r[2], r[3]);
  hi = make_uint4(r[4], r[5], r[6], r[7]);
}
__device__ __forceinline__ void scale4(uint4& u, __half2 f) {
  __half2* h = reinterpret_cast<__half2*>(&u);
#pragma unroll
  for (int i = 0; i < 4; ++i) h[i] = __hmul2(h[i], f);
}
__device__ __forceinline__ void put16(uint32_t addr, const uint4& u) {
  asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(addr), "r"(u.x), "r"(u.y), "r"(u.z), "r"(u.w) : "memory");
}

// the bits of 32 positions from t on that a row sees
__device__ __forceinline__ uint32_t below(int n) { return n <= 0 ? 0u : n >= 32 ? ~0u : (1u << n) - 1u; }
__device__ __forceinline__ uint32_t seen32(const TreeArgs& a, const Portion& p, int i, int first, int t) {
  if (a.mask == nullptr) return below(p.p0 + i + 1 - t) & ~below(first - t);
  uint32_t bits = below(p.p0 - t) & ~below(first - t);
  const int j = t - p.p0;                                          // the drafted token at t
  if (j > -32 && j < p.n) {
    const unsigned long long* m = a.mask + (long long)(p.row + i) * a.words;
    uint32_t d;
    if (j < 0) {
      d = (uint32_t)(m[0] << -j);
    } else {
      unsigned long long w = m[j >> 6] >> (j & 63);
      if ((j & 63) > 32 && (j >> 6) + 1 < a.words) w |= m[(j >> 6) + 1] << (64 - (j & 63));
      d = (uint32_t)w;
    }
    bits |= d & below(p.n - j) & ~below(-j);
  }
  return bits;
}

__device__ __forceinline__ void put8(uint32_t addr, const uint2& u) { asm volatile("st.shared.v2.b32 [%0], {%1,%2};" ::"r"(addr), "r"(u.x), "r"(u.y) : "memory"); }
__device__ __forceinline__ void softmax_sync() { asm volatile("bar.sync 1, 256;" ::: "memory"); }      // the eight softmax warps
__device__ __forceinline__ float max3(float a, float b, float c) {
  float y;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
  return y;
}
// REF, as an exponent: of the largest finite scale of `n` <= 64 positions, two of them a lane.  Not below LEAST_SCALE: a weight / scale is at most 2^(15 + 80), whose sums stay finite
// (with 2^-107, which a head of zeros is stored with, 2^14 of them did not, and what came behind them was lost)
__device__ __forceinline__ void ask_ref(const float* scale, int n, uint32_t (&u)[2]) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int x = 0; x < 2; ++x) u[x] = x * 32 + lane < n ? __float_as_uint(__ldcg(scale + x * 32 + lane)) : 0u;
}
__device__ __forceinline__ int ref_of(const uint32_t (&u)[2]) {
  const uint32_t top = __reduce_max_sync(0xffffffffu, max(u[0] < 0x7f800000u ? u[0] : 0u, u[1] < 0x7f800000u ? u[1] : 0u));   // (not a negative one either)
  return top >= 0x00800000u ? min(max((int)(top >> 23) - 127, -80), 100) : 0;
}
__device__ __forceinline__ float pow2(int e) { return __uint_as_float((uint32_t)(127 + e) << 23); }      // -126 <= e <= 127

template <int DIM, int VDIM, int KIND, bool PAIR>
__global__ void __launch_bounds__(THREADS, 1) tree_attn_tc_kernel(const __grid_constant__ TreeArgs a, int* __restrict__ timeouts) {
  using C = Tc<DIM, VDIM, KIND, PAIR>;
  constexpr bool BITS8 = C::BITS8;
  constexpr int TILE = PAIR ? 2 * ROWS : ROWS, STAGES = C::STAGES;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t smem = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* smem_gen = smem_raw + (smem - smem_u32(smem_raw));
  const uint32_t queries = smem + STAGES * C::STAGE;               // [groups' own rows][DIM]
  Tail& sm = *reinterpret_cast<Tail*>(smem_gen + STAGES * C::STAGE + C::ALL_Q);
  const int warp = __shfl_sync(0xffffffffu, (int)threadIdx.x >> 5, 0), lane = threadIdx.x & 31;

  pdl_launch_dependents();
  pdl_wait();
  Portion p = portion_of(a, blockIdx.z);
  if (!p.held) {
    if (a.splits == 1 && blockIdx.y == 0) nan_rows<VDIM>(a, p);
    return;
  }
  // (known to be the same in all lanes, so that what the products' instructions take needs no moves to uniform registers)
  p.slot = __shfl_sync(0xffffffffu, p.slot, 0), p.p0 = __shfl_sync(0xffffffffu, p.p0, 0), p.row = __shfl_sync(0xffffffffu, p.row, 0), p.n = __shfl_sync(0xffffffffu, p.n, 0);
  const int g = blockIdx.y % a.G, R = p.n * a.rep, tiles = (R + TILE - 1) / TILE, tile = tiles - 1 - (int)blockIdx.y / a.G, r0 = tile * TILE;   // (the last ones see most)
  if (tile < 0) return;
  const int groups = !PAIR || r0 + ROWS < R ? 2 : 1;               // (with one the second has no rows and no blocks)

  if (threadIdx.x == 0) {
    sm.dead = 0;
    for (int i = 0; i < STAGES; ++i) {
      mbar_init(smem_u32(&sm.full[i]), LOADERS / 32);
      mbar_init(smem_u32(&sm.empty[i]), 1);
    }
    for (int i = 0; i < 2; ++i) {
      for (int x = 0; x < 2; ++x) {
        mbar_init(smem_u32(&sm.s_full[i][x]), 1);
        mbar_init(smem_u32(&sm.p_full[i][x]), 4);
      }
      mbar_init(smem_u32(&sm.o_done[i]), 1);
    }
    mbar_init(smem_u32(&sm.q_full), 8);
    mbar_init(smem_u32(&sm.drain), 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == ISSUER) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sm.tmem)), "r"(512u) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tcgen05_fence_before();
  __syncthreads();
  tcgen05_fence_after();
  const uint32_t tmem = __shfl_sync(0xffffffffu, sm.tmem, 0);
  volatile int* dead = &sm.dead;

  // ---- which keys
  const int i0 = r0 / a.rep, i1 = min(p.n - 1, (r0 + TILE - 1) / a.rep);
  int near = i0, far = i1;
  if (a.depth != nullptr && a.window < 1 << 30) {                  // (without a window depths do not matter)
    near = 1 << 29;
    far = 0;
    for (int i = i0 + lane; i <= i1; i += 32) {
      const int d = depth_of(a, p, i);
      near = min(near, d);
      far = max(far, d);
    }
    near = __reduce_min_sync(0xffffffffu, near);
    far = __reduce_max_sync(0xffffffffu, far);
  }
  const int lo = first_key(a, p, near), hi = end_key(a, p, i1), all_lo = first_key(a, p, far), all_hi = a.mask != nullptr ? p.p0 : p.p0 + i0 + 1;
  const int nb = (hi - lo + KEYS - 1) / KEYS, b0 = __shfl_sync(0xffffffffu, (int)((long long)nb * blockIdx.x / a.splits), 0),
            n = __shfl_sync(0xffffffffu, (int)((long long)nb * (blockIdx.x + 1) / a.splits), 0) - b0;
  const int start = lo + b0 * KEYS;

  if (warp < 8) {
    // ================================================================ softmax
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(SOFTMAX_REGS));
    const int s = warp >> 2, w = warp & 3, r = w * 32 + lane;
    const int row = r0 + (PAIR ? s * ROWS : 0) + r;
    const bool there = row < R, warp_there = row - lane < R;
    const int i = there ? row / a.rep : p.n - 1, h = there ? g * a.rep + row - i * a.rep : g * a.rep;
    const uint32_t lanes = tmem + ((uint32_t)(w * 32) << 16);
    uint32_t scales[2] = {0u, 0u};
    if constexpr (BITS8) ask_ref(a.v.scale_at(p.slot, g) + start, n > 0 ? min(hi - start, KEYS) : 0, scales);
    // ---- queries go to shared memory, a row a warp at a time, and what a row's products are multiplied by to sm.row_f
    constexpr int SHARE = TILE / 8;
    const int c4 = lane * 4, place = BITS8 ? place_of<DIM>(c4 >> 4, (c4 >> 3) & 1) + (c4 & 7) : c4;     // a lane's four channels, and where they go
    const uint32_t lane_at = queries + (place >> 6) * C::Q_SLAB + (place & 7) * 2;
    const int chunk = (place & 63) >> 3;
    const float factor_all = a.scale * (a.softcap > 0.f ? 1.f : LOG2E);
    int rr = warp * SHARE, qi = (r0 + rr) / a.rep, qh = r0 + rr - qi * a.rep;                            // the row in the tile, its token and its head of the group's
#pragma unroll 1
    for (int x0 = 0; x0 < SHARE && (r0 + rr) / 32 * 32 < R; x0 += 8) {                                  // (warps without a row need none)
      uint2 u[8];
      float f[8];
#pragma unroll
      for (int x = 0; x < 8; ++x) {
        const bool in = r0 + rr + x < R;
        u[x] = in && lane < DIM / 4 ? *reinterpret_cast<const uint2*>(a.q + (long long)(p.row + qi) * a.ldq + (g * a.rep + qh) * DIM + c4) : make_uint2(0u, 0u);
        f[x] = a.temp != nullptr && in ? a.temp[g * a.rep + qh] * factor_all : factor_all;
        if (++qh == a.rep) {
          qh = 0;
          ++qi;
        }
      }
#pragma unroll
      for (int x = 0; x < 8; ++x, ++rr) {
        const bool flip = f[x] < 0.f;                              // (so that the largest product is the largest score)
        uint2 w;
        if constexpr (BITS8) {
          const uint32_t m = __vmaxu2(u[x].x & 0x7fff7fffu, u[x].y & 0x7fff7fffu);
          const Down down = down_of(__reduce_max_sync(0xffffffffu, max(m & 0xffffu, m >> 16)));
          const float by = flip ? -down.by : down.by;
          float y[4];
          unpack_bf16x2(u[x].x, y[0], y[1]);
          unpack_bf16x2(u[x].y, y[2], y[3]);
          w = make_uint2(pack_f16x2(y[0] * by, y[1] * by), pack_f16x2(y[2] * by, y[3] * by));
          f[x] *= down.back;
        } else {
          const uint32_t sign = flip ? 0x80008000u : 0u;
          w = make_uint2(u[x].x ^ sign, u[x].y ^ sign);
        }
        if (lane < DIM / 4) put8(lane_at + (PAIR ? (rr >> 7) * C::Q_BYTES : 0) + (rr & 127) * 128 + ((chunk ^ (rr & 7)) << 4), w);
        if (lane == 0) sm.row_f[rr] = fabsf(f[x]);
      }
    }
    fence_proxy_async_smem();
    __syncwarp();
    if (lane == 0) mbar_arrive(smem_u32(&sm.q_full));
    softmax_sync();
    const float rf = sm.row_f[PAIR ? s * ROWS + r : r];
    const int first = first_key(a, p, depth_of(a, p, i));
    const float two_by_cap = a.softcap > 0.f ? 2.f * LOG2E / a.softcap : 0.f;
    const uint32_t values = lanes + VALUES + s * 128;
    float m = -1e30f, l = 0.f;
    bool alive = true;
    int done = 0;                                                  // of the group's blocks
    const int ref = BITS8 ? ref_of(scales) : 0;
    const float ref_l = (float)ref, ref_inv = pow2(-ref);
    // (a row's first block sees to a maximum; -1e30 stands for none, so that nothing is less than it but -inf)
#pragma unroll 1
    for (int j = PAIR ? 0 : s; j < n && s < groups; j += PAIR ? 1 : 2, ++done) {
      const int st = j % STAGES, buf = done & 1;
      const uint32_t scores = lanes + s * 128 + buf * KEYS;
      float4 k4[BITS8 ? 4 : 1];                                    // a quarter of the keys' scales, asked for together
      auto ask_scales = [&](int half) {
#pragma unroll
        for (int c = 0; c < (BITS8 ? 4 : 0); ++c) k4[c] = *reinterpret_cast<const float4*>(&sm.ks[st][half * 16 + c * 4]);
      };
      if constexpr (BITS8) {
        if (!(alive = warp_wait(smem_u32(&sm.full[st]), (j / STAGES) & 1, dead))) break;
        ask_scales(0);
      }
      if (!(alive = warp_wait(smem_u32(&sm.s_full[s][buf]), (done >> 1) & 1, dead))) break;
      tcgen05_fence_after();
      float keep = 1.f;
      bool moved = false;
      if (warp_there) {
        uint32_t v[KEYS];
        tmem_ld32(scores, v);
        tmem_ld32(scores + 32, v + 32);
        tmem_ld_wait();
        if constexpr (BITS8) {
#pragma unroll
          for (int half = 0; half < 4; ++half) {
            float4 f4[4];
#pragma unroll
            for (int c = 0; c < 4; ++c) f4[c] = k4[c];
            if (half < 3) ask_scales(half + 1);
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              const int x = half * 16 + c * 4;
              float a0, a1;
              unpack2(mul2(pack2(__uint_as_float(v[x]), __uint_as_float(v[x + 1])), pack2(f4[c].x, f4[c].y)), a0, a1);
              v[x] = __float_as_uint(a0);
              v[x + 1] = __float_as_uint(a1);
              unpack2(mul2(pack2(__uint_as_float(v[x + 2]), __uint_as_float(v[x + 3])), pack2(f4[c].z, f4[c].w)), a0, a1);
              v[x + 2] = __float_as_uint(a0);
              v[x + 3] = __float_as_uint(a1);
            }
          }
        }
        const int t = start + j * KEYS;
        const bool odd = BITS8 && sm.odd[st] != 0;
        float factor = rf, add = ref_l;                            // x = v * factor + add, in powers of two (with the values' scales)
        if (odd || a.softcap > 0.f) {
          factor = 1.f;
          add = 0.f;
        }
        auto each = [&](auto with) {                               // with(pair of products with their keys' scales, column of the first)
#pragma unroll
          for (int c = 0; c < KEYS; c += 2) {
            float x0, x1;
            unpack2(with(pack2(__uint_as_float(v[c]), __uint_as_float(v[c + 1])), c), x0, x1);
            v[c] = __float_as_uint(x0);
            v[c + 1] = __float_as_uint(x1);
          }
        };
        if (a.softcap > 0.f) {
          each([&](f32x2 x, int c) {
            float x0, x1;
            unpack2(mul2(x, both(rf)), x0, x1);
            return fma2(pack2(capped(x0, a.softcap, two_by_cap), capped(x1, a.softcap, two_by_cap)), both(LOG2E), BITS8 ? pack2(sm.lv[st][c], sm.lv[st][c + 1]) : both(0.f));
          });
        } else if (odd) {
          each([&](f32x2 x, int c) { return fma2(x, both(rf), pack2(sm.lv[st][c], sm.lv[st][c + 1])); });
        }
        if (t < all_lo || t + KEYS > min(all_hi, hi)) {
#pragma unroll
          for (int c = 0; c < KEYS; c += 32) {
            const uint32_t bits = seen32(a, p, i, first, t + c) & below(hi - t - c);
#pragma unroll
            for (int e = 0; e < 32; ++e)
              if (!((bits >> e) & 1u)) v[c + e] = 0xff800000u;
          }
        }
        float tops[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int c = 0; c < KEYS; c += 8)
#pragma unroll
          for (int e = 0; e < 4; ++e) tops[e] = max3(tops[e], __uint_as_float(v[c + 2 * e]), __uint_as_float(v[c + 2 * e + 1]));
        const float top = fmaf(fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3])), factor, add);
        // ---- the maximum moves for rows that have outgrown it
        const bool grown = top - m > SLACK;
        moved = __any_sync(0xffffffffu, grown);
        if (moved) {
          const float to = grown ? top : m;
          keep = grown ? ex2(m - to) : 1.f;
          m = to;
          l *= keep;
        }
        const f32x2 by = both(factor), off = both(add + C::LIFT - m);
        // ---- weights
        f32x2 sum = 0ull;
#pragma unroll
        for (int c = 0; c < KEYS; c += 16) {
          uint32_t hi16[8], lo16[8];
#pragma unroll
          for (int e = 0; e < 16; e += 4) {
            float w0, w1, w2, w3;
            unpack2(fma2(pack2(__uint_as_float(v[c + e]), __uint_as_float(v[c + e + 1])), by, off), w0, w1);
            unpack2(fma2(pack2(__uint_as_float(v[c + e + 2]), __uint_as_float(v[c + e + 3])), by, off), w2, w3);
            w0 = ex2(w0);
            w1 = ex2(w1);
            w2 = ex2(w2);
            w3 = ex2(w3);
            sum = add2(sum, add2(pack2(w0, w1), pack2(w2, w3)));
            if constexpr (BITS8) {
              hi16[e / 2] = pack_f16x2(w0, w1);
              hi16[e / 2 + 1] = pack_f16x2(w2, w3);
              v[c + e] = __float_as_uint(w0);
              v[c + e + 1] = __float_as_uint(w1);
              v[c + e + 2] = __float_as_uint(w2);
              v[c + e + 3] = __float_as_uint(w3);
            } else {
              float x0, x1;
              hi16[e / 2] = pack_bf16x2(w0, w1);
              unpack_bf16x2(hi16[e / 2], x0, x1);
              lo16[e / 2] = pack_bf16x2(w0 - x0, w1 - x1);
              hi16[e / 2 + 1] = pack_bf16x2(w2, w3);
              unpack_bf16x2(hi16[e / 2 + 1], x0, x1);
              lo16[e / 2 + 1] = pack_bf16x2(w2 - x0, w3 - x1);
            }
          }
          tmem_st8(scores + c / 2, hi16);
          if constexpr (!BITS8) tmem_st8(scores + 32 + c / 2, lo16);
        }
        float s0, s1;
        if (odd) {                                                 // p = weight / what is left of the scale
          sum = 0ull;
#pragma unroll
          for (int c = 0; c < KEYS; c += 4) {
            const float4 r4 = *reinterpret_cast<const float4*>(&sm.rv[st][c]);
            sum = fma2(pack2(__uint_as_float(v[c]), __uint_as_float(v[c + 1])), pack2(r4.x, r4.y), sum);
            sum = fma2(pack2(__uint_as_float(v[c + 2]), __uint_as_float(v[c + 3])), pack2(r4.z, r4.w), sum);
          }
        }
        unpack2(sum, s0, s1);
        l = fmaf(s0 + s1, odd ? 1.f : ref_inv, l);
      }
      // The products of the group's last block are waited for every time, so that no phase of theirs is missed (two later, it would look like one that has yet to come)
      if (done > 0) {
        if (!(alive = warp_wait(smem_u32(&sm.o_done[s]), (done - 1) & 1, dead))) break;
        if (moved) {
          tcgen05_fence_after();
#pragma unroll 1
          for (int c = 0; c < VDIM; c += 16) {
            uint32_t o[16];
            tmem_ld16(values + c, o);
            tmem_ld_wait();
#pragma unroll
            for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * keep);
            tmem_st16(values + c, o);
          }
        }
      }
      tmem_st_wait();
      tcgen05_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&sm.p_full[s][buf]));
    }
    if (alive && done > 0) alive = warp_wait(smem_u32(&sm.o_done[s]), (done - 1) & 1, dead);
    if (!alive) l = __uint_as_float(0x7fc00000u);
    tcgen05_fence_after();
    // ---- groups of the same rows meet: the second's by way of shared memory, where the keys were (both groups' last products are done, and with them the loads)
    float* other = reinterpret_cast<float*>(smem_gen);             // [VDIM][ROWS], a row's channels a thread's own
    float top = m, sum = l, f0 = n > 0 ? 1.f : 0.f, f1 = 0.f;
    const bool two = !PAIR && n > 1;
    if constexpr (!PAIR) {
      softmax_sync();
      if (s == 1) {
        sm.ml[r] = make_float2(m, l);
        if (two) {
#pragma unroll 1
          for (int c = 0; c < VDIM; c += 32) {
            uint32_t o[32];
            tmem_ld32(values + c, o);
            tmem_ld_wait();
#pragma unroll
            for (int e = 0; e < 32; ++e) other[(c + e) * ROWS + r] = __uint_as_float(o[e]);
          }
        }
      }
      softmax_sync();
      const float2 ml = sm.ml[r];
      top = fmaxf(m, ml.x);
      f0 = n > 0 ? ex2(m - top) : 0.f;
      f1 = two ? ex2(ml.x - top) : 0.f;
      sum = l * f0 + ml.y * f1;                                    // (NaN if a wait ran out)
      if (isnan(l) || isnan(ml.y)) sum = l + ml.y;
    }
    if ((PAIR || s == 0) && warp_there) {
      const long long rows = (long long)a.M * a.H, at = (long long)(p.row + i) * a.H + h;
      const bool whole = a.splits == 1, wide = reinterpret_cast<uintptr_t>(a.out) % 16 == 0;       // (rows are whole 16-byte vectors; where they begin may be on an 8-byte boundary)
      const float inv = whole ? 1.f / sum : 1.f;
      float probe = 0.f;
#pragma unroll 1
      for (int c = 0; c < VDIM; c += 32) {
        uint32_t o[32];
        if (n > 0) {
          tmem_ld32(values + c, o);
          tmem_ld_wait();
        }
#pragma unroll
        for (int e = 0; e < 32; e += 8) {
          float y[8];
#pragma unroll
          for (int x = 0; x < 8; ++x) {
            y[x] = n > 0 ? __uint_as_float(o[e + x]) * f0 : 0.f;
            if (two) y[x] = fmaf(other[(c + e + x) * ROWS + r], f1, y[x]);
            y[x] *= inv;
            probe = fmaf(y[x], 0.f, probe);
          }
          const int col = c + e, ch = BITS8 && VDIM == 128 ? (col & 63) / 8 * 16 + (col >> 6) * 8 : col;
          if (there) {
            if (whole) {
              const uint4 u = pack8(y);
              bf16* dst = a.out + at * VDIM + ch;
              if (wide) {
                *reinterpret_cast<uint4*>(dst) = u;
              } else {
                reinterpret_cast<uint2*>(dst)[0] = make_uint2(u.x, u.y);
                reinterpret_cast<uint2*>(dst)[1] = make_uint2(u.z, u.w);
              }
            } else {
              float4* dst = reinterpret_cast<float4*>(a.ws + (blockIdx.x * rows + at) * VDIM + ch);
              dst[0] = make_float4(y[0], y[1], y[2], y[3]);
              dst[1] = make_float4(y[4], y[5], y[6], y[7]);
            }
          }
        }
      }
      if (!whole) {
        if (there) reinterpret_cast<float2*>(a.ws + a.splits * rows * VDIM)[blockIdx.x * rows + at] = make_float2(top, sum);
      } else {                                                     // rows with numbers that are not finite, or without a key
        unsigned again = __ballot_sync(0xffffffffu, there && !(probe == 0.f));
        while (again) {
          const int src = __ffs(again) - 1;
          again &= again - 1;
          const int ii = __shfl_sync(0xffffffffu, i, src), hh = __shfl_sync(0xffffffffu, h, src);
          float y[VDIM / 32];
          form_again<DIM, VDIM, KIND>(a, p, ii, hh, y);
          for (int c = 0; c < VDIM / 32; ++c) a.out[((long long)(p.row + ii) * a.H + hh) * VDIM + c * 32 + lane] = __float2bfloat16_rn(y[c]);
        }
      }
    }
    tcgen05_fence_before();
  } else if (warp < ISSUER) {
    // ================================================================ keys and values
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(LOADER_REGS));
    const int th = threadIdx.x - 256, kt = th % C::KT, vt = th % C::VT, k0 = th / C::KT, v0 = th / C::VT;
    constexpr int KSTEP = LOADERS / C::KT, VSTEP = LOADERS / C::VT;                            // a lane's keys are so far apart
    // the lane's places in the next block to ask for
    const uint8_t *kp = a.k.at(p.slot, start + k0, g) + kt * 16, *vp = a.v.at(p.slot, start + v0, g) + vt * 16;
    const float *ksp = BITS8 ? a.k.scale_at(p.slot, g) + start : nullptr, *vsp = BITS8 ? a.v.scale_at(p.slot, g) + start : nullptr;
    uint32_t scales[2] = {0u, 0u};
    uint4 kr[C::AHEAD][C::KN], vr[C::AHEAD][C::VN];
    float ks[C::AHEAD], vs[C::AHEAD][C::VN];                       // of key th < 64, and of the lane's values
    auto ask = [&](int j, int x) {
      if (j >= n) return;
      const int left = hi - start - j * KEYS;                      // keys from the block's first on
      if (left >= KEYS) {
#pragma unroll
        for (int c = 0; c < C::KN; ++c) kr[x][c] = ldg_act(kp + c * KSTEP * a.k.pos);
#pragma unroll
        for (int c = 0; c < C::VN; ++c) vr[x][c] = ldg_act(vp + c * VSTEP * a.v.pos);
        if constexpr (BITS8) {
          if (th < KEYS) ks[x] = __ldcg(ksp + th);
#pragma unroll
          for (int c = 0; c < C::VN; ++c) vs[x][c] = __ldcg(vsp + v0 + c * VSTEP);
        }
      } else {
#pragma unroll
        for (int c = 0; c < C::KN; ++c) kr[x][c] = k0 + c * KSTEP < left ? ldg_act(kp + c * KSTEP * a.k.pos) : make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
        for (int c = 0; c < C::VN; ++c) vr[x][c] = v0 + c * VSTEP < left ? ldg_act(vp + c * VSTEP * a.v.pos) : make_uint4(0u, 0u, 0u, 0u);
        if constexpr (BITS8) {
          if (th < KEYS) ks[x] = th < left ? __ldcg(ksp + th) : 0.f;
#pragma unroll
          for (int c = 0; c < C::VN; ++c) vs[x][c] = v0 + c * VSTEP < left ? __ldcg(vsp + v0 + c * VSTEP) : -1.f;     // (none)
        }
      }
      kp += KEYS * a.k.pos;
      vp += KEYS * a.v.pos;
      if constexpr (BITS8) {
        ksp += KEYS;
        vsp += KEYS;
      }
    };
    // where the lane's vectors go: the second half of 16 codes beside the first or in the next slab, the vectors of other keys some rows of 128 bytes on
    auto place = [&](int key, int tid, int wide) {
      const int p0 = BITS8 ? (wide == 128 ? place_of<128>(tid, 0) : place_of<64>(tid, 0)) : tid * 8;
      return (uint32_t)((p0 >> 6) * C::SLAB + key * 128 + ((((p0 & 63) >> 3) ^ (key & 7)) << 4));
    };
    const uint32_t k_at = place(k0, kt, DIM), v_at = C::K_BYTES + place(v0, vt, VDIM);
    auto put = [&](uint32_t at, bool wide, const uint4& x, const uint4& y) {
      put16(at, x);
      put16(wide ? at + C::SLAB : at ^ 16u, y);                    // (of 64 channels they are neighbours, which the swizzle keeps in one pair)
    };
#pragma unroll
    for (int x = 0; x < C::AHEAD; ++x) ask(x, x);
    if constexpr (BITS8) ask_ref(a.v.scale_at(p.slot, g) + start, n > 0 ? min(hi - start, KEYS) : 0, scales);
    const int ref = BITS8 ? ref_of(scales) : 0;
    const float ref_inv = pow2(-ref);
    bool alive = true;
#pragma unroll 1
    for (int j0 = 0; j0 < n && alive; j0 += C::AHEAD) {
#pragma unroll
      for (int x = 0; x < C::AHEAD; ++x) {
        const int j = j0 + x, st = j % STAGES;
        if (j >= n) break;
        if (!(alive = warp_wait(smem_u32(&sm.empty[st]), ((j / STAGES) & 1) ^ 1u, dead))) break;
        const uint32_t at = smem + st * C::STAGE;
        if constexpr (BITS8) {
#pragma unroll
          for (int c = 0; c < C::KN; ++c) {
            uint4 lo16, hi16;
            widen<KIND>(kr[x][c], lo16, hi16);
            put(at + k_at + c * KSTEP * 128, DIM == 128, lo16, hi16);
          }
          if (th < KEYS) sm.ks[st][th] = ks[x];
          bool odd = false;
#pragma unroll
          for (int c = 0; c < C::VN; ++c) {
            uint4 lo16, hi16;
            widen<KIND>(vr[x][c], lo16, hi16);
            const float f = vs[x][c] * ref_inv;
            const bool near = (f >= 0x1p-8f && f < 64.f) || vs[x][c] == -1.f;
            odd |= !near;
            const __half2 f2 = __float2half2_rn(near ? f : 1.f);
            scale4(lo16, f2);                                      // (zeros, where there is none)
            scale4(hi16, f2);
            put(at + v_at + c * VSTEP * 128, VDIM == 128, lo16, hi16);
            if (vt == 0) {
              const float y = near ? pow2(ref) : max_nan(vs[x][c], LEAST_SCALE);
              sm.lv[st][v0 + c * VSTEP] = lg2(y);
              sm.rv[st][v0 + c * VSTEP] = __fdividef(1.f, y);
            }
          }
          odd = __any_sync(0xffffffffu, odd);
          if (lane == 0) reinterpret_cast<uint8_t*>(&sm.odd[st])[warp - 8] = odd;
        } else {
#pragma unroll
          for (int c = 0; c < C::KN; ++c) put16(at + k_at + c * KSTEP * 128, kr[x][c]);
#pragma unroll
          for (int c = 0; c < C::VN; ++c) put16(at + v_at + c * VSTEP * 128, vr[x][c]);
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&sm.full[st]));
        ask(j + C::AHEAD, x);
      }
    }
  } else {
    // ================================================================ products
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(OTHER_REGS));
    if (warp == ISSUER) {
      const uint32_t one = elect_one();
      constexpr uint32_t types = BITS8 ? 0u : (1u << 7) | (1u << 10);
      constexpr uint32_t idesc_qk = (1u << 4) | types | ((uint32_t)(KEYS >> 3) << 17) | ((uint32_t)(ROWS >> 4) << 24);
      constexpr uint32_t idesc_pv = (1u << 4) | types | (1u << 16) | ((uint32_t)(VDIM >> 3) << 17) | ((uint32_t)(ROWS >> 4) << 24);      // (the values lie with the keys as rows)
      bool alive = n > 0 && warp_wait(smem_u32(&sm.q_full), 0, dead);
      auto scores = [&](int j, int s, int done) {                  // of group s's block number `done`
        const int st = j % STAGES, buf = done & 1;
        if (!warp_wait(smem_u32(&sm.full[st]), (j / STAGES) & 1, dead)) return false;
        tcgen05_fence_after();
        const uint32_t at = smem + st * C::STAGE, q = queries + (PAIR ? s * C::Q_BYTES : 0);
#pragma unroll
        for (int k = 0; k < DIM / 16; ++k)
          mma_if(one, tmem + s * 128 + buf * KEYS, make_smem_desc(q + (k >> 2) * C::Q_SLAB + (k & 3) * 32), make_smem_desc(at + (k >> 2) * C::SLAB + (k & 3) * 32), idesc_qk, k > 0);
        commit_if(one, smem_u32(&sm.s_full[s][buf]));
        return true;
      };
      auto weighted = [&](int j, int s, int done) {
        const int st = j % STAGES, buf = done & 1;
        if (!warp_wait(smem_u32(&sm.p_full[s][buf]), (done >> 1) & 1, dead)) return false;
        tcgen05_fence_after();
        const uint32_t at = smem + st * C::STAGE + C::K_BYTES;
#pragma unroll
        for (int part = 0; part < (BITS8 ? 1 : 2); ++part)
#pragma unroll
          for (int k = 0; k < KEYS / 16; ++k)
            mma_tmem_a_if(one, tmem + VALUES + s * 128, tmem + s * 128 + buf * KEYS + part * 32 + k * 8, make_smem_desc_mn(at + k * 16 * 128, C::SLAB), idesc_pv,
                          done > 0 || part > 0 || k > 0);
        return true;
      };
      // A group's scores come behind the products with the weights whose place they take, a block ahead of its softmax
      if constexpr (PAIR) {
        for (int s = 0; s < groups && alive; ++s) alive = scores(0, s, 0);
#pragma unroll 1
        for (int j = 0; j < n && alive; ++j) {
          for (int s = 0; s < groups && alive && j + 1 < n; ++s) alive = scores(j + 1, s, j + 1);
          for (int s = 0; s < groups && alive; ++s) {
            if (!(alive = weighted(j, s, j))) break;
            commit_if(one, smem_u32(&sm.o_done[s]));
            if (s == groups - 1) commit_if(one, smem_u32(&sm.empty[j % STAGES]));
          }
        }
      } else {
        for (int j = 0; j < 3 && j < n && alive; ++j) alive = scores(j, j & 1, j >> 1);
#pragma unroll 1
        for (int j = 0; j < n && alive; ++j) {
          if (j + 3 < n && !(alive = scores(j + 3, (j + 3) & 1, (j + 3) >> 1))) break;
          if (!(alive = weighted(j, j & 1, j >> 1))) break;
          commit_if(one, smem_u32(&sm.empty[j % STAGES]));
          commit_if(one, smem_u32(&sm.o_done[j & 1]));
        }
      }
    }
  }

  // ---- products in flight end before the memory that they use is given back
  if (__syncthreads_or(*dead)) {
    if (threadIdx.x == 0) atomicAdd_system(timeouts, 1);
    if (warp == ISSUER) {
      commit_if(elect_one(), smem_u32(&sm.drain));
      wait_in_flight(smem_u32(&sm.drain), 0u);
    }
  }
  tcgen05_fence_before();
  __syncthreads();
  if (warp == ISSUER) {
    tcgen05_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
  }
}

template <int DIM, int VDIM, int KIND, bool PAIR> int launch(const TreeArgs& a, int nseg, cudaStream_t stream) {
  using C = Tc<DIM, VDIM, KIND, PAIR>;
  constexpr int SMEM = C::STAGES * C::STAGE + C::ALL_Q + (int)sizeof(Tail) + 1024;
  static_assert(SMEM <= 232448 && C::STAGES * C::STAGE >= ROWS * VDIM * 4 && C::STAGES >= 4, "shared memory");
  static bool configured[64] = {};                                 // per device
  int dev = 0;
  LIA_CUDA(cudaGetDevice(&dev));
  if (dev >= 64 || !configured[dev]) {
    LIA_CUDA(cudaFuncSetAttribute(tree_attn_tc_kernel<DIM, VDIM, KIND, PAIR>, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM));
    if (dev < 64) configured[dev] = true;
  }
  static const bool split_fits = [] {                              // the registers that the warps trade must be those that the block gets
    cudaFuncAttributes at{};
    return cudaFuncGetAttributes(&at, tree_attn_tc_kernel<DIM, VDIM, KIND, PAIR>) == cudaSuccess && at.numRegs == LAUNCH_REGS;
  }();
  LIA_CHECK_ARG(split_fits, "lia_tree_attn: the kernel was built with too few registers");
  int* timeouts = lia_formed_again_word();
  LIA_CHECK_ARG(timeouts, "lia_tree_attn: no memory for the count of waits that ran out");
  LIA_CUDA(lia_launch(tree_attn_tc_kernel<DIM, VDIM, KIND, PAIR>, dim3(a.splits, a.tiles * a.G, nseg), dim3(THREADS), SMEM, stream, a, timeouts));
  return LIA_OK;
}
template <int DIM, int VDIM, int KIND> int launch_rows(const TreeArgs& a, int rows, int nseg, cudaStream_t stream) {
  return rows > ROWS ? launch<DIM, VDIM, KIND, true>(a, nseg, stream) : launch<DIM, VDIM, KIND, false>(a, nseg, stream);
}
template <int KIND> int launch_dims(const TreeArgs& a, int rows, int nseg, cudaStream_t stream) {
  if (a.k.dim == 128) return a.v.dim == 128 ? launch_rows<128, 128, KIND>(a, rows, nseg, stream) : launch_rows<128, 64, KIND>(a, rows, nseg, stream);
  return a.v.dim == 128 ? launch_rows<64, 128, KIND>(a, rows, nseg, stream) : launch_rows<64, 64, KIND>(a, rows, nseg, stream);
}

}  // namespace

// blocks of `rows` rows, 128 or 256 (a.tiles of them a portion); parts of split histories are left in a.ws
int lia_tree_attn_tc(const void* args, int type, int rows, int nseg, lia_stream_t stream_) {
  const TreeArgs& a = *reinterpret_cast<const TreeArgs*>(args);
  cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_);
  switch (type) {
    case LIA_CACHE_BF16: return launch_dims<LIA_CACHE_BF16>(a, rows, nseg, stream);
    case LIA_CACHE_INT8: return launch_dims<LIA_CACHE_INT8>(a, rows, nseg, stream);
    default: return launch_dims<LIA_CACHE_E4M3>(a, rows, nseg, stream);
  }
}
