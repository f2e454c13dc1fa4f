// Attention of drafted tokens (tree_attn.cu has the formulas) for many rows of a key head: 128 rows of (token, head) to a block, on tcgen05.
//
//   warps 0-3, 4-7   two groups that take the history's blocks of 64 keys in turn, each with a maximum, a sum and weighted values of its own; a thread has one row, which is one
//                    lane of TMEM.  They meet at the end.
//   warps 8-15       bring keys and values: 16 bytes a lane from memory, 8-bit codes as fp16, into shared memory as the products want them (128-byte swizzle).  Positions behind the last key
//                    become zeros, so that nothing unwritten is multiplied.
//   warp 16          the products (three more are there for their registers)
// TMEM, 512 columns: group s has its scores at 64 s, in their place its weights (fp16, or two bf16 parts), and its weighted values at 128 + 128 s; the queries, from where
// they are the products' first operand, lie at QUERIES: shared memory, which takes 128 bytes a clock, is left to keys and values.
// The weighted values stay in TMEM from block to block.  Weights are relative to a maximum that moves only when a row has exceeded it by 2^8 (they fit fp16 up to there); only then
// its group multiplies what it has, behind the products of its last block.
//
// What bounds it at 128 rows: the powers (one a score, 16 a clock and SM: 1024 clocks for 128 keys of 128 rows) as well as the tensor cores (1024 with 8-bit codes, 1536 with bf16 and its two
// parts of weights); with fewer rows memory (1400 clocks for 128 keys of 8 bits, 2800 of bf16).
#include "pairs.cuh"
#include "tree_attn.cuh"
#include "umma.cuh"

int* lia_timeout_word();                                           // moe_sm100.cu

namespace {

constexpr int ROWS = 128, KEYS = 64, THREADS = 640, LOADERS = 256, ISSUER = 16;
constexpr int SOFTMAX_REGS = 128, LOADER_REGS = 96, OTHER_REGS = 24; // of a thread, by what its four warps do (setmaxnreg: multiples of 8); the launch gives 96
constexpr uint32_t VALUES = 128, QUERIES = 384;
constexpr float SLACK = 8.f;                                       // how far, in powers of two, weights may exceed 1

template <int DIM, int VDIM, int KIND>
struct Tc {
  static constexpr bool BITS8 = KIND != LIA_CACHE_BF16;
  static constexpr int SLAB = KEYS * 128;                          // 64 channels of 16 bits of a block's keys
  static constexpr int K_BYTES = DIM / 64 * SLAB, V_BYTES = VDIM / 64 * SLAB, STAGE = K_BYTES + V_BYTES;
  static constexpr int STAGES = 196608 / STAGE > 8 ? 8 : 196608 / STAGE;
  static constexpr int KT = DIM * (BITS8 ? 1 : 2) / 16, VT = VDIM * (BITS8 ? 1 : 2) / 16;      // lanes of a key, of a value
  static constexpr int KN = KEYS * KT / LOADERS, VN = KEYS * VT / LOADERS;                       // vectors of a lane
  static constexpr int AHEAD = BITS8 ? 4 : 2;                      // blocks on their way from memory
  static constexpr float LIFT = BITS8 ? 7.f : 0.f;                 // weights are 2^(x - maximum + LIFT): below 2^15 in fp16
};
struct Tail {
  float ks[8][KEYS], lv[8][KEYS], rv[8][KEYS];                     // of a stage's keys: scale; of its values: log2 of the scale, its inverse
  float2 ml[ROWS];
  uint64_t full[8], empty[8], s_full[2], p_full[2], o_done[2], q_full, drain;
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

template <int DIM, int VDIM, int KIND>
__global__ void __launch_bounds__(THREADS, 1) tree_attn_tc_kernel(const TreeArgs a, int* __restrict__ timeouts) {
  using C = Tc<DIM, VDIM, KIND>;
  constexpr bool BITS8 = C::BITS8;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t smem = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* smem_gen = smem_raw + (smem - smem_u32(smem_raw));
  Tail& sm = *reinterpret_cast<Tail*>(smem_gen + C::STAGES * C::STAGE);
  const int warp = __shfl_sync(0xffffffffu, (int)threadIdx.x >> 5, 0), lane = threadIdx.x & 31;

  pdl_launch_dependents();
  pdl_wait();
  const Portion p = portion_of(a, blockIdx.z);
  if (!p.held) {
    if (a.splits == 1 && blockIdx.y == 0) nan_rows<VDIM>(a, p);
    return;
  }
  const int g = blockIdx.y % a.G, R = p.n * a.rep, tiles = (R + ROWS - 1) / ROWS, tile = tiles - 1 - (int)blockIdx.y / a.G, r0 = tile * ROWS;   // (the last ones see most)
  if (tile < 0) return;

  if (threadIdx.x == 0) {
    sm.dead = 0;
    for (int i = 0; i < C::STAGES; ++i) {
      mbar_init(smem_u32(&sm.full[i]), LOADERS / 32);
      mbar_init(smem_u32(&sm.empty[i]), 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(smem_u32(&sm.s_full[i]), 1);
      mbar_init(smem_u32(&sm.p_full[i]), 4);
      mbar_init(smem_u32(&sm.o_done[i]), 1);
    }
    mbar_init(smem_u32(&sm.q_full), 4);
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
  const int i0 = r0 / a.rep, i1 = min(p.n - 1, (r0 + ROWS - 1) / a.rep);
  int near = i0, far = i1;
  if (a.depth != nullptr) {
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
  const int nb = (hi - lo + KEYS - 1) / KEYS, b0 = (int)((long long)nb * blockIdx.x / a.splits), n = (int)((long long)nb * (blockIdx.x + 1) / a.splits) - b0;
  const int start = lo + b0 * KEYS;

  if (warp < 8) {
    // ================================================================ softmax
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(SOFTMAX_REGS));
    const int s = warp >> 2, w = warp & 3, r = w * 32 + lane;
    const bool there = r0 + r < R, warp_there = r0 + w * 32 < R;
    const int i = there ? (r0 + r) / a.rep : p.n - 1, h = there ? g * a.rep + (r0 + r) - i * a.rep : g * a.rep;
    const uint32_t lanes = tmem + ((uint32_t)(w * 32) << 16);
    float rf = a.scale * (a.temp != nullptr ? a.temp[h] : 1.f) * (a.softcap > 0.f ? 1.f : LOG2E);
    const bool flip = rf < 0.f;                                    // (so that the largest product is the largest score)
    {                                                              // queries: group 0's go to TMEM, both know their factor
      const bf16* src = a.q + (long long)(p.row + i) * a.ldq + h * DIM;
      uint32_t top = 0;
      uint2 u[DIM / 4];
#pragma unroll
      for (int c = 0; c < DIM / 4; ++c) {
        u[c] = there ? *reinterpret_cast<const uint2*>(src + c * 4) : make_uint2(0u, 0u);
        top = max(top, max(max(u[c].x & 0x7fffu, (u[c].x >> 16) & 0x7fffu), max(u[c].y & 0x7fffu, (u[c].y >> 16) & 0x7fffu)));
      }
      const Down down = down_of(top);
      const float by = flip ? -down.by : down.by;
      if constexpr (BITS8) rf *= down.back;
      rf = fabsf(rf);
      if (s == 0) {
#pragma unroll
        for (int c0 = 0; c0 < DIM / 2; c0 += 16) {                 // 32 numbers of a row
          uint32_t q[16];
#pragma unroll
          for (int e = 0; e < 8; ++e) {                            // four of them
            if constexpr (BITS8) {
              const int at = c0 * 2 + e * 4, c = DIM == 128 ? (at & 63) / 8 * 16 + (at >> 6) * 8 + (at & 7) : at;
              float x[4];
              unpack_bf16x2(u[c / 4].x, x[0], x[1]);
              unpack_bf16x2(u[c / 4].y, x[2], x[3]);
              q[2 * e] = pack_f16x2(x[0] * by, x[1] * by);
              q[2 * e + 1] = pack_f16x2(x[2] * by, x[3] * by);
            } else {
              const uint32_t sign = flip ? 0x80008000u : 0u;
              q[2 * e] = u[c0 / 2 + e].x ^ sign;
              q[2 * e + 1] = u[c0 / 2 + e].y ^ sign;
            }
          }
          tmem_st16(lanes + QUERIES + c0, q);
        }
        tmem_st_wait();
        tcgen05_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&sm.q_full));
      }
    }
    const int first = first_key(a, p, depth_of(a, p, i));
    const float two_by_cap = a.softcap > 0.f ? 2.f * LOG2E / a.softcap : 0.f;
    const uint32_t scores = lanes + s * KEYS, values = lanes + VALUES + s * 128;
    float m = -INFINITY, l = 0.f;
    bool alive = true;
    int done = 0;                                                  // of the group's blocks
#pragma unroll 1
    for (int j = s; j < n; j += 2, ++done) {
      const int st = j % C::STAGES;
      if constexpr (BITS8)
        if (!(alive = warp_wait(smem_u32(&sm.full[st]), (j / C::STAGES) & 1, dead))) break;
      if (!(alive = warp_wait(smem_u32(&sm.s_full[s]), done & 1, dead))) break;
      tcgen05_fence_after();
      if (warp_there) {
        uint32_t v[KEYS];
        tmem_ld32(scores, v);
        tmem_ld32(scores + 32, v + 32);
        tmem_ld_wait();
        const int t = start + j * KEYS;
        // ---- scores in powers of two (with the values' scales)
        auto scaled = [&](auto with) {                             // with(pair of products times the row's factor, log2 of the values' scales)
#pragma unroll
          for (int c = 0; c < KEYS; c += 4) {
            float4 k4 = make_float4(1.f, 1.f, 1.f, 1.f), l4 = make_float4(0.f, 0.f, 0.f, 0.f);
            if constexpr (BITS8) {
              k4 = *reinterpret_cast<const float4*>(&sm.ks[st][c]);
              l4 = *reinterpret_cast<const float4*>(&sm.lv[st][c]);
            }
            f32x2 x = pack2(__uint_as_float(v[c]), __uint_as_float(v[c + 1])), y = pack2(__uint_as_float(v[c + 2]), __uint_as_float(v[c + 3]));
            if constexpr (BITS8) {
              x = mul2(x, pack2(k4.x, k4.y));
              y = mul2(y, pack2(k4.z, k4.w));
            }
            x = with(x, pack2(l4.x, l4.y));
            y = with(y, pack2(l4.z, l4.w));
            float x0, x1;
            unpack2(x, x0, x1);
            v[c] = __float_as_uint(x0);
            v[c + 1] = __float_as_uint(x1);
            unpack2(y, x0, x1);
            v[c + 2] = __float_as_uint(x0);
            v[c + 3] = __float_as_uint(x1);
          }
        };
        if (a.softcap > 0.f) {
          scaled([&](f32x2 x, f32x2 lv) {
            float x0, x1;
            unpack2(mul2(x, both(rf)), x0, x1);
            return fma2(pack2(capped(x0, a.softcap, two_by_cap), capped(x1, a.softcap, two_by_cap)), both(LOG2E), lv);
          });
        } else if constexpr (BITS8) {
          scaled([&](f32x2 x, f32x2 lv) { return fma2(x, both(rf), lv); });
        } else {
          scaled([&](f32x2 x, f32x2) { return mul2(x, both(rf)); });
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
        for (int c = 0; c < KEYS; ++c) tops[c & 3] = fmaxf(tops[c & 3], __uint_as_float(v[c]));
        const float top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
        // ---- the maximum moves for rows that have outgrown it
        const bool grown = top > m + SLACK || (m == -INFINITY && top != -INFINITY);
        if (__any_sync(0xffffffffu, grown)) {
          const float to = grown ? top : m, keep = grown ? ex2(m - to) : 1.f;
          m = to;
          l *= keep;
          if (done > 0) {
            if (!(alive = warp_wait(smem_u32(&sm.o_done[s]), (done - 1) & 1, dead))) break;
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
        const float off = C::LIFT - (m == -INFINITY ? 0.f : m);
        // ---- weights
        f32x2 sum = 0ull;
#pragma unroll
        for (int c = 0; c < KEYS; c += 16) {
          uint32_t hi16[8], lo16[8];
#pragma unroll
          for (int e = 0; e < 16; e += 4) {
            float w0, w1, w2, w3;
            unpack2(add2(pack2(__uint_as_float(v[c + e]), __uint_as_float(v[c + e + 1])), both(off)), w0, w1);
            unpack2(add2(pack2(__uint_as_float(v[c + e + 2]), __uint_as_float(v[c + e + 3])), both(off)), w2, w3);
            w0 = ex2(w0);
            w1 = ex2(w1);
            w2 = ex2(w2);
            w3 = ex2(w3);
            if constexpr (BITS8) {
              const float4 r4 = *reinterpret_cast<const float4*>(&sm.rv[st][c + e]);
              sum = fma2(pack2(w0, w1), pack2(r4.x, r4.y), sum);
              sum = fma2(pack2(w2, w3), pack2(r4.z, r4.w), sum);
              hi16[e / 2] = pack_f16x2(w0, w1);
              hi16[e / 2 + 1] = pack_f16x2(w2, w3);
            } else {
              sum = add2(sum, add2(pack2(w0, w1), pack2(w2, w3)));
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
        unpack2(sum, s0, s1);
        l += s0 + s1;
        tmem_st_wait();
        tcgen05_fence_before();
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&sm.p_full[s]));
    }
    if (alive && done > 0) alive = warp_wait(smem_u32(&sm.o_done[s]), (done - 1) & 1, dead);
    if (!alive) l = __uint_as_float(0x7fc00000u);
    tcgen05_fence_after();
    // ---- the groups' rows meet: the second's by way of shared memory, where the keys were (both groups' last products are done, and with them the loads)
    auto groups_sync = [] { asm volatile("bar.sync 1, 256;" ::: "memory"); };
    float* other = reinterpret_cast<float*>(smem_gen);             // [VDIM][ROWS], a row's channels a thread's own
    groups_sync();
    if (s == 1) {
      sm.ml[r] = make_float2(m, l);
      if (n > 1) {
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
    groups_sync();
    if (s == 0 && warp_there) {
      const float2 ml = sm.ml[r];
      const float top = fmaxf(m, ml.x), base = top == -INFINITY ? 0.f : top, f0 = n > 0 ? ex2(m - base) : 0.f, f1 = n > 1 ? ex2(ml.x - base) : 0.f;
      const float sum = l * f0 + ml.y * f1;                        // (NaN if a wait ran out)
      const long long rows = (long long)a.M * a.H, at = (long long)(p.row + i) * a.H + h;
      const bool whole = a.splits == 1;
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
            if (n > 1) y[x] = fmaf(other[(c + e + x) * ROWS + r], f1, y[x]);
            y[x] *= inv;
            probe = fmaf(y[x], 0.f, probe);
          }
          const int col = c + e, ch = BITS8 && VDIM == 128 ? (col & 63) / 8 * 16 + (col >> 6) * 8 : col;
          if (there) {
            if (whole) {
              *reinterpret_cast<uint4*>(a.out + at * VDIM + ch) = pack8(y);
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
    const int th = threadIdx.x - 256, kt = th % C::KT, vt = th % C::VT;
    const uint8_t *kbase = a.k.at(p.slot, 0, g) + kt * 16, *vbase = a.v.at(p.slot, 0, g) + vt * 16;
    const float* scales = BITS8 && th < 2 * KEYS ? (th < KEYS ? a.k.scale_at(p.slot, g) : a.v.scale_at(p.slot, g)) : nullptr;
    uint4 kr[C::AHEAD][C::KN], vr[C::AHEAD][C::VN];
    float sc[C::AHEAD];
    auto ask = [&](int j, int x) {
      const int t = start + j * KEYS;
#pragma unroll
      for (int c = 0; c < C::KN; ++c) {
        const int key = t + th / C::KT + c * (LOADERS / C::KT);
        kr[x][c] = j < n && key < hi ? ldg_act(kbase + (long long)key * a.k.pos) : make_uint4(0u, 0u, 0u, 0u);
      }
#pragma unroll
      for (int c = 0; c < C::VN; ++c) {
        const int key = t + th / C::VT + c * (LOADERS / C::VT);
        vr[x][c] = j < n && key < hi ? ldg_act(vbase + (long long)key * a.v.pos) : make_uint4(0u, 0u, 0u, 0u);
      }
      if constexpr (BITS8)
        if (th < 2 * KEYS) sc[x] = j < n && t + (th & (KEYS - 1)) < hi ? __ldcg(scales + t + (th & (KEYS - 1))) : 1.f;
    };
    auto put = [&](uint32_t tile_at, int key, int tid, int wide, const uint4& u) {
      if constexpr (BITS8) {
        uint4 x, y;
        widen<KIND>(u, x, y);
        const int p0 = wide == 128 ? place_of<128>(tid, 0) : place_of<64>(tid, 0), p1 = wide == 128 ? place_of<128>(tid, 1) : place_of<64>(tid, 1);
        put16(tile_at + (p0 >> 6) * C::SLAB + key * 128 + ((((p0 & 63) >> 3) ^ (key & 7)) << 4), x);
        put16(tile_at + (p1 >> 6) * C::SLAB + key * 128 + ((((p1 & 63) >> 3) ^ (key & 7)) << 4), y);
      } else {
        put16(tile_at + (tid >> 3) * C::SLAB + key * 128 + (((tid & 7) ^ (key & 7)) << 4), u);
      }
    };
#pragma unroll
    for (int x = 0; x < C::AHEAD; ++x) ask(x, x);
    bool alive = true;
#pragma unroll 1
    for (int j0 = 0; j0 < n && alive; j0 += C::AHEAD) {
#pragma unroll
      for (int x = 0; x < C::AHEAD; ++x) {
        const int j = j0 + x, st = j % C::STAGES;
        if (j >= n) break;
        if (!(alive = warp_wait(smem_u32(&sm.empty[st]), ((j / C::STAGES) & 1) ^ 1u, dead))) break;
        const uint32_t at = smem + st * C::STAGE;
#pragma unroll
        for (int c = 0; c < C::KN; ++c) put(at, th / C::KT + c * (LOADERS / C::KT), kt, DIM, kr[x][c]);
#pragma unroll
        for (int c = 0; c < C::VN; ++c) put(at + C::K_BYTES, th / C::VT + c * (LOADERS / C::VT), vt, VDIM, vr[x][c]);
        if constexpr (BITS8) {
          if (th < KEYS) {
            sm.ks[st][th] = sc[x];
          } else if (th < 2 * KEYS) {
            const float y = max_nan(sc[x], LEAST_SCALE);
            sm.lv[st][th - KEYS] = lg2(y);
            sm.rv[st][th - KEYS] = __fdividef(1.f, y);
          }
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
      auto scores = [&](int j) {
        const int st = j % C::STAGES;
        if (!warp_wait(smem_u32(&sm.full[st]), (j / C::STAGES) & 1, dead)) return false;
        tcgen05_fence_after();
        const uint32_t at = smem + st * C::STAGE;
#pragma unroll
        for (int k = 0; k < DIM / 16; ++k) mma_tmem_a_if(one, tmem + (j & 1) * KEYS, tmem + QUERIES + k * 8, make_smem_desc(at + (k >> 2) * C::SLAB + (k & 3) * 32), idesc_qk, k > 0);
        commit_if(one, smem_u32(&sm.s_full[j & 1]));
        return true;
      };
      if (alive) alive = scores(0);
      if (alive && n > 1) alive = scores(1);
#pragma unroll 1
      for (int j = 0; j < n && alive; ++j) {
        const int st = j % C::STAGES, s = j & 1;
        if (!(alive = warp_wait(smem_u32(&sm.p_full[s]), (j >> 1) & 1, dead))) break;
        tcgen05_fence_after();
        const uint32_t at = smem + st * C::STAGE + C::K_BYTES;
#pragma unroll
        for (int part = 0; part < (BITS8 ? 1 : 2); ++part)
#pragma unroll
          for (int k = 0; k < KEYS / 16; ++k)
            mma_tmem_a_if(one, tmem + VALUES + s * 128, tmem + s * KEYS + part * 32 + k * 8, make_smem_desc_mn(at + k * 16 * 128, C::SLAB), idesc_pv, j > 1 || part > 0 || k > 0);
        commit_if(one, smem_u32(&sm.empty[st]));
        commit_if(one, smem_u32(&sm.o_done[s]));
        if (j + 2 < n) alive = scores(j + 2);
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

template <int DIM, int VDIM, int KIND> int launch(const TreeArgs& a, int nseg, cudaStream_t stream) {
  using C = Tc<DIM, VDIM, KIND>;
  constexpr int SMEM = C::STAGES * C::STAGE + (int)sizeof(Tail) + 1024;
  static_assert(SMEM <= 232448 && C::STAGES * C::STAGE >= ROWS * VDIM * 4, "shared memory");
  static bool configured[64] = {};                                 // per device
  int dev = 0;
  LIA_CUDA(cudaGetDevice(&dev));
  if (dev >= 64 || !configured[dev]) {
    LIA_CUDA(cudaFuncSetAttribute(tree_attn_tc_kernel<DIM, VDIM, KIND>, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM));
    if (dev < 64) configured[dev] = true;
  }
  static const bool split_fits = [] {                              // the registers that the warps trade must be those that the block gets
    cudaFuncAttributes at{};
    return cudaFuncGetAttributes(&at, tree_attn_tc_kernel<DIM, VDIM, KIND>) == cudaSuccess && at.numRegs * THREADS >= 128 * (2 * SOFTMAX_REGS + 2 * LOADER_REGS + OTHER_REGS);
  }();
  LIA_CHECK_ARG(split_fits, "lia_tree_attn: the kernel was built with too few registers");
  int* timeouts = lia_timeout_word();
  LIA_CHECK_ARG(timeouts, "lia_tree_attn: no memory for the count of waits that ran out");
  LIA_CUDA(lia_launch_after(tree_attn_tc_kernel<DIM, VDIM, KIND>, dim3(a.splits, a.tiles * a.G, nseg), dim3(THREADS), SMEM, stream, a, timeouts));
  return LIA_OK;
}
template <int KIND> int launch_dims(const TreeArgs& a, int nseg, cudaStream_t stream) {
  if (a.k.dim == 128) return a.v.dim == 128 ? launch<128, 128, KIND>(a, nseg, stream) : launch<128, 64, KIND>(a, nseg, stream);
  return a.v.dim == 128 ? launch<64, 128, KIND>(a, nseg, stream) : launch<64, 64, KIND>(a, nseg, stream);
}

}  // namespace

// blocks of 128 rows (a.tiles of them a portion); parts of split histories are left in a.ws
int lia_tree_attn_tc(const void* args, int type, int nseg, lia_stream_t stream_) {
  const TreeArgs& a = *reinterpret_cast<const TreeArgs*>(args);
  cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_);
  switch (type) {
    case LIA_CACHE_BF16: return launch_dims<LIA_CACHE_BF16>(a, nseg, stream);
    case LIA_CACHE_INT8: return launch_dims<LIA_CACHE_INT8>(a, nseg, stream);
    default: return launch_dims<LIA_CACHE_E4M3>(a, nseg, stream);
  }
}
