// Attention of portions of new tokens -- a decoded token, a chain or a tree of drafted ones, a part of a prompt -- behind their cached histories, over caches of bf16, int8 or e4m3 (and,
// by way of tree_attn_4bit.cu, of 4 bits).
//
//   s_ij = cap tanh(temp_h scale ks_j (q_i . k_j) / cap),   o_i = sum_j p_ij vs_j v_j / sum_j p_ij,   p_ij = e^(s_ij - max) over the j that row i sees
//
// Few rows see a long history: what counts is that the history is read once, whatever the number of rows and of query heads that share a key head.  So a block has up to 32 of the
// portion's (token, head) rows of one key head, its four warps take 16 keys each in turn, and the history is split over as many blocks as fill the GPU: up to eight of them are a cluster and
// read one another's sums, more leave theirs in a workspace for a second launch.  (With the workspace for these too, a token each of 16 sequences behind 1901 positions took 27 us instead of 23.)
//
// The keys are the rows of a product (16 of them) and the queries its columns (8), so that one token of up to eight query heads wastes little.  Keys and values go
// from memory to the lanes that multiply them, without shared memory between: a product sums over channels in any order, so a lane's 16 neighbouring bytes of a key
// are four steps' operands, and a product's rows may be any channels, so the 16 neighbouring bytes of a value are its operands for 16 (bf16: 8) of them.  Weights come out of the
// first product with keys along rows and go into the second with keys along the sum: eight by eight of them are transposed across the warp (movmatrix).
//
// 8-bit codes are exact in fp16 and so are multiplied there: q goes to fp16 by a power of two of its own for each row (its 8 bits fit; what is 2^-29 of the row's largest is
// less exact), a key's scale is multiplied into its scores, and a value's into its weight -- in the exponent, x = s + log2 vs, so that the maximum bounds the product and no scale is
// too large or small: weights are 2^(x - max + 7) in fp16, 11 bits (fewer below 2^-21 of the row's largest, none below 2^-32), and their sum takes p = weight / vs in fp32.  With bf16 caches weights are two bf16 parts: 16 bits.
// The maximum moves only when a key exceeds it by 2^8, which the 7 leaves room for; the rows' sums are multiplied only then.
//
// Bound: bf16 caches by memory, 8-bit ones by instructions too (a byte is widened, half of them after two codes change places; a score takes some fifteen).  A token of 16 heads on 8 for each of 16
// histories of 60000 positions: bf16 563 us (7.0 TB/s; a copy, which writes half of what it moves, has 6.55), int8 398 to 419 (5.1 to 4.8), e4m3 377 to 391 (5.4 to 5.2).  Behind 1901 positions, int8: 19.5 us, of which memory 10; the rest is
// one block's way from its first load to its last sum.  (Arguments are taken where the launch put them: copied to each thread's stack, for rows that are formed again, they cost 2 us a block.)
#include "mma.cuh"
#include "tree_attn.cuh"

int lia_tree_attn_tc(const void* args, int type, int rows, int nseg, lia_stream_t stream);      // tree_attn_sm100.cu
int lia_tree_attn_4bit(const void* args, int nr, int nseg, lia_stream_t stream);                // tree_attn_4bit.cu

namespace {

constexpr int MAX_SPLITS = 64;

// blocks of an SM, by the registers that the rows' sums and the keys and values on their way take
constexpr int blocks_an_sm(int kind, int nr) { return kind == LIA_CACHE_INT4 ? tree_attn4_blocks(nr) : nr == 1 ? (kind == LIA_CACHE_BF16 ? 3 : 4) : nr == 2 ? (kind == LIA_CACHE_BF16 ? 2 : 3) : 2; }

template <int DIM, int VDIM, int KIND, int NR>
struct Shape {
  static constexpr bool BITS8 = KIND != LIA_CACHE_BF16;
  static constexpr int STEPS = DIM / 16;                           // products of a block of 16 keys with 8 rows' queries
  static constexpr int MT = VDIM / 16;                             // products of 16 channels of a block's values with 8 rows' weights
  static constexpr int KV = DIM * (BITS8 ? 1 : 2) / 64;            // 16-byte vectors of a key in a lane
  static constexpr int VB = VDIM * (BITS8 ? 1 : 2) / 8;            // bytes of a value in a lane
  static constexpr int ROWS = 8 * NR;
  static constexpr int Q_BYTES = NR * STEPS * 32 * 8, O_BYTES = WARPS * ROWS * VDIM * 4, BIG = Q_BYTES > O_BYTES ? Q_BYTES : O_BYTES;
  static constexpr int SMEM = BIG + ROWS * 4 + WARPS * ROWS * 8;
  static constexpr float LIFT = BITS8 ? 7.f : 0.f;                 // a weight of the maximum is 2^LIFT, one that is just not outgrown 2^15 in fp16
  // the channel of the first of a lane's pair in the i-th product with the values
  static __device__ __forceinline__ int channel(int i, int gq) { return BITS8 ? gq * (VDIM / 8) + 2 * i : (i >> 2) * 64 + gq * 8 + (i & 3) * 2; }
};
template <int DIM, int VDIM, int KIND, int NR>
__global__ void __launch_bounds__(THREADS, blocks_an_sm(KIND, NR)) tree_attn_kernel(const __grid_constant__ TreeArgs a) {
  using S = Shape<DIM, VDIM, KIND, NR>;
  constexpr bool BITS8 = S::BITS8;
  constexpr int RQ = BITS8 ? 1 : 2;
  extern __shared__ uint4 smem[];
  float* row_f = reinterpret_cast<float*>(reinterpret_cast<uint8_t*>(smem) + S::BIG);        // [ROWS] what a row's products with keys are multiplied by
  float2* part = reinterpret_cast<float2*>(row_f + S::ROWS);       // [WARPS][ROWS] maximum, sum
  uint2* qs = reinterpret_cast<uint2*>(smem);                      // [NR][STEPS][32]
  pdl_launch_dependents();
  pdl_wait();
  const Portion p = portion_of(a, blockIdx.z);
  if (!p.held) {
    if (a.splits <= CLUSTER && blockIdx.x == 0 && blockIdx.y == 0) nan_rows<VDIM>(a, p);
    return;
  }
  const int warp = __shfl_sync(0xffffffffu, (int)threadIdx.x >> 5, 0), lane = threadIdx.x & 31, gq = lane >> 2, t4 = lane & 3;   // (known to be the same in all lanes)
  const int tile = blockIdx.y / a.G, g = blockIdx.y - tile * a.G, r0 = tile * S::ROWS, R = p.n * a.rep;
  if (r0 >= R) return;

  // ---- which keys
  const int i0 = r0 / a.rep, i1 = min(p.n - 1, (r0 + S::ROWS - 1) / a.rep);
  int near = i0, far = i1;                                         // depths of the block's tokens
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
  const int lo = first_key(a, p, near), hi = end_key(a, p, i1), all_lo = first_key(a, p, far), all_hi = min(hi, a.mask != nullptr ? p.p0 : p.p0 + i0 + 1);
  const int nb = (hi - lo + 15) >> 4, b0 = (int)((long long)nb * blockIdx.x / a.splits), b1 = (int)((long long)nb * (blockIdx.x + 1) / a.splits);

  const uint8_t *kbase = a.k.at(p.slot, 0, g) + t4 * 16, *vbase = a.v.at(p.slot, 0, g) + gq * (BITS8 ? S::VB : 16);
  const float *ksc = BITS8 ? a.k.scale_at(p.slot, g) : nullptr, *vsc = BITS8 ? a.v.scale_at(p.slot, g) : nullptr;
  uint4 kr[2][S::KV];                                              // keys gq and gq + 8
  uint32_t vr[4][S::VB / 4];                                       // values 2 t4, 2 t4 + 1, 8 + 2 t4, 9 + 2 t4
  float ks[2], vs[2];                                              // of keys gq and gq + 8
  auto load_k = [&](int b) {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int key = min(lo + b * 16 + j * 8 + gq, hi - 1);
      const uint8_t* src = kbase + (long long)key * a.k.pos;
#pragma unroll
      for (int c = 0; c < S::KV; ++c) kr[j][c] = ldg_act(src + c * 64);
      if constexpr (BITS8) {
        ks[j] = __ldcg(ksc + key);
        vs[j] = __ldcg(vsc + key);
      }
    }
  };
  auto load_v = [&](int b) {
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const uint8_t* src = vbase + (long long)min(lo + b * 16 + (c >> 1) * 8 + t4 * 2 + (c & 1), hi - 1) * a.v.pos;
      if constexpr (S::VB == 8) {
        const uint2 u = __ldcg(reinterpret_cast<const uint2*>(src));
        vr[c][0] = u.x;
        vr[c][1] = u.y;
      } else {
#pragma unroll
        for (int w = 0; w < S::VB / 16; ++w) *reinterpret_cast<uint4*>(&vr[c][w * 4]) = ldg_act(src + w * 128);
      }
    }
  };

  if (b0 + warp < b1) {                                            // (on their way while the queries are brought: chains of 8 behind 280 119 -> 113 us)
    load_k(b0 + warp);
    load_v(b0 + warp);
  }

  // ---- queries: rows (token, head) in the order of the products' operands
  for (int r = warp; r < S::ROWS; r += WARPS) {
    const bool there = r0 + r < R;
    const int i = (r0 + r) / a.rep, h = g * a.rep + (r0 + r) - i * a.rep;
    uint2 u = make_uint2(0u, 0u);
    if (there && lane < DIM / 4) u = *reinterpret_cast<const uint2*>(a.q + (p.row + i) * a.ldq + h * DIM + lane * 4);
    float f = a.scale * (a.temp != nullptr && there ? a.temp[h] : 1.f) * (a.softcap > 0.f ? 1.f : LOG2E);
    uint2 w = u;
    if constexpr (BITS8) {
      uint32_t top = max(max((u.x & 0x7fffu), (u.x >> 16) & 0x7fffu), max((u.y & 0x7fffu), (u.y >> 16) & 0x7fffu));
      const Down down = down_of(__reduce_max_sync(0xffffffffu, top));
      float x[4];
      unpack_bf16x2(u.x, x[0], x[1]);
      unpack_bf16x2(u.y, x[2], x[3]);
      w = make_uint2(pack_f16x2(x[0] * down.by, x[1] * down.by), pack_f16x2(x[2] * down.by, x[3] * down.by));
      f *= down.back;
    }
    if (lane < DIM / 4) {                                          // four neighbouring channels are a lane's operand of one step
      const int c = lane * 4, t = BITS8 ? (c >> 4) & 3 : (c >> 3) & 3, step = BITS8 ? (c >> 6) * 4 + ((c >> 2) & 3) : (c >> 5) * 2 + ((c >> 2) & 1);
      qs[((r >> 3) * S::STEPS + step) * 32 + (r & 7) * 4 + t] = w;
    }
    if (lane == 0) row_f[r] = f;
  }
  __syncthreads();
  uint2 qa[NR <= RQ ? NR : 1][NR <= RQ ? S::STEPS : 1];            // few rows' queries stay in registers, the others' in shared memory
  if constexpr (NR <= RQ) {
#pragma unroll
    for (int r = 0; r < NR; ++r)
#pragma unroll
      for (int s = 0; s < S::STEPS; ++s) qa[r][s] = qs[(r * S::STEPS + s) * 32 + lane];
  }

  float rf[NR][2], m[NR][2], l[NR][2];                             // of the lane's rows 2 t4 and 2 t4 + 1 of every eight
#pragma unroll
  for (int r = 0; r < NR; ++r)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      rf[r][e] = row_f[r * 8 + t4 * 2 + e];
      m[r][e] = NONE;
      l[r][e] = 0.f;
    }
  float o[NR][S::MT][4];                                           // [..][0]: a lane's first channel of a pair and row 2 t4, [1]: row 2 t4 + 1, [2], [3]: its second channel
#pragma unroll
  for (int r = 0; r < NR; ++r)
#pragma unroll
    for (int n = 0; n < S::MT; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[r][n][e] = 0.f;

  const float two_by_cap = a.softcap > 0.f ? 2.f * LOG2E / a.softcap : 0.f;
#pragma unroll 1
  for (int b = b0 + warp; b < b1; b += WARPS) {
    // ---- products of 16 keys and all rows: s[r][0], [1]: key gq and rows 2 t4, 2 t4 + 1; [2], [3]: key gq + 8
    float s[NR][4];
#pragma unroll
    for (int r = 0; r < NR; ++r)
#pragma unroll
      for (int e = 0; e < 4; ++e) s[r][e] = 0.f;
#pragma unroll
    for (int st = 0; st < S::STEPS; ++st) {
      uint32_t ka[4];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        if constexpr (BITS8) {
          const uint4& u = kr[j][st >> 2];
          uint32_t w = (st & 3) == 0 ? u.x : (st & 3) == 1 ? u.y : (st & 3) == 2 ? u.z : u.w;
          if constexpr (KIND == LIA_CACHE_INT8) {
            w ^= 0x80808080u;
            ka[j] = int8x2(__byte_perm(w, 0x64646464u, 0x4140));
            ka[2 + j] = int8x2(__byte_perm(w, 0x64646464u, 0x4342));
          } else {
            ka[j] = e4m3x2(w & 0xffffu);
            ka[2 + j] = e4m3x2(w >> 16);
          }
        } else {
          const uint4& u = kr[j][st >> 1];
          ka[j] = st & 1 ? u.z : u.x;
          ka[2 + j] = st & 1 ? u.w : u.y;
        }
      }
#pragma unroll
      for (int r = 0; r < NR; ++r) {
        uint2 q;
        if constexpr (NR <= RQ) q = qa[r][st];
        else q = qs[(r * S::STEPS + st) * 32 + lane];
        if constexpr (BITS8) mma_f16(s[r], ka, q.x, q.y);
        else mma_bf16(s[r], ka, q.x, q.y);
      }
    }
    float kf[2] = {1.f, 1.f}, lv[2] = {0.f, 0.f}, rv[2] = {1.f, 1.f};
    if constexpr (BITS8) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        kf[j] = ks[j];
        const float y = max_nan(vs[j], LEAST_SCALE);
        lv[j] = lg2(y);
        rv[j] = __fdividef(1.f, y);
      }
    }
    if (b + WARPS < b1) load_k(b + WARPS);
    // ---- scores, as powers of two and with the values' scales
    const int key0 = lo + b * 16;
    if (a.softcap > 0.f) {
#pragma unroll
      for (int r = 0; r < NR; ++r)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[r][e] = fmaf(capped(s[r][e] * kf[e >> 1] * rf[r][e & 1], a.softcap, two_by_cap), LOG2E, lv[e >> 1]);
    } else {
#pragma unroll
      for (int r = 0; r < NR; ++r)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[r][e] = BITS8 ? fmaf(s[r][e] * kf[e >> 1], rf[r][e & 1], lv[e >> 1]) : s[r][e] * rf[r][e & 1];
    }
    if (key0 < all_lo || key0 + 16 > all_hi) {
#pragma unroll
      for (int r = 0; r < NR; ++r)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int i = min((r0 + r * 8 + t4 * 2 + e) / a.rep, p.n - 1), d = depth_of(a, p, i);
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const int t = key0 + j * 8 + gq;
            if (t >= hi || !sees(a, p, i, d, t)) s[r][j * 2 + e] = -INFINITY;
          }
        }
    }
    // ---- the maximum (m: less LIFT) moves only for rows that have outgrown it
    bool grown = false;
#pragma unroll
    for (int r = 0; r < NR; ++r)
#pragma unroll
      for (int e = 0; e < 4; ++e) grown |= s[r][e] - m[r][e & 1] > SLACK + S::LIFT;
    if (__any_sync(0xffffffffu, grown)) {
#pragma unroll
      for (int r = 0; r < NR; ++r)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float top = fmaxf(s[r][e], s[r][2 + e]);
#pragma unroll
          for (int x = 4; x < 32; x <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
          const bool up = top - m[r][e] > SLACK + S::LIFT;
          const float keep = up ? ex2(m[r][e] - (top - S::LIFT)) : 1.f;
          if (up) m[r][e] = top - S::LIFT;
          l[r][e] *= keep;
#pragma unroll
          for (int n = 0; n < S::MT; ++n) {
            o[r][n][e] *= keep;
            o[r][n][2 + e] *= keep;
          }
        }
    }
    // ---- weights, turned into the products' other operand
    uint32_t pb[BITS8 ? 1 : 2][NR][2];
#pragma unroll
    for (int r = 0; r < NR; ++r) {
      float w[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        w[e] = ex2(s[r][e] - m[r][e & 1]);
        l[r][e & 1] = BITS8 ? fmaf(w[e], rv[e >> 1], l[r][e & 1]) : l[r][e & 1] + w[e];
      }
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        if constexpr (BITS8) {
          pb[0][r][j] = transposed(pack_f16x2(w[2 * j], w[2 * j + 1]));
        } else {
          const uint32_t hi2 = pack_bf16x2(w[2 * j], w[2 * j + 1]);
          float x, y;
          unpack_bf16x2(hi2, x, y);
          pb[0][r][j] = transposed(hi2);
          pb[BITS8 ? 0 : 1][r][j] = transposed(pack_bf16x2(w[2 * j] - x, w[2 * j + 1] - y));
        }
      }
    }
    // ---- weighted values
#pragma unroll
    for (int w = 0; w < S::VB / 4; ++w) {
      constexpr int PER = BITS8 ? 4 : 2;                           // channels of a word
      uint32_t va[PER][2];
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const uint32_t u0 = vr[2 * c][w], u1 = vr[2 * c + 1][w];
        if constexpr (BITS8) {
          uint32_t x = __byte_perm(u0, u1, 0x5140), y = __byte_perm(u0, u1, 0x7362);
          if constexpr (KIND == LIA_CACHE_INT8) {
            x ^= 0x80808080u;
            y ^= 0x80808080u;
            va[0][c] = int8x2(__byte_perm(x, 0x64646464u, 0x4140));
            va[1][c] = int8x2(__byte_perm(x, 0x64646464u, 0x4342));
            va[2][c] = int8x2(__byte_perm(y, 0x64646464u, 0x4140));
            va[3][c] = int8x2(__byte_perm(y, 0x64646464u, 0x4342));
          } else {
            va[0][c] = e4m3x2(x & 0xffffu);
            va[1][c] = e4m3x2(x >> 16);
            va[2][c] = e4m3x2(y & 0xffffu);
            va[3][c] = e4m3x2(y >> 16);
          }
        } else {
          va[0][c] = __byte_perm(u0, u1, 0x5410);
          va[1][c] = __byte_perm(u0, u1, 0x7632);
        }
      }
#pragma unroll
      for (int c = 0; c < PER; c += 2) {
        const uint32_t v4[4] = {va[c][0], va[c + 1][0], va[c][1], va[c + 1][1]};
        const int n = (w * PER + c) >> 1;
#pragma unroll
        for (int r = 0; r < NR; ++r) {
          if constexpr (BITS8) {
            mma_f16(o[r][n], v4, pb[0][r][0], pb[0][r][1]);
          } else {
            mma_bf16(o[r][n], v4, pb[0][r][0], pb[0][r][1]);
            mma_bf16(o[r][n], v4, pb[BITS8 ? 0 : 1][r][0], pb[BITS8 ? 0 : 1][r][1]);
          }
        }
      }
    }
    if (b + WARPS < b1) load_v(b + WARPS);
  }

  // ---- the warps' parts meet in shared memory
  __syncthreads();                                                 // (queries have been read)
  float* os = reinterpret_cast<float*>(smem);
#pragma unroll
  for (int r = 0; r < NR; ++r)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      float x = l[r][e];
#pragma unroll
      for (int d = 4; d < 32; d <<= 1) x += __shfl_xor_sync(0xffffffffu, x, d);
      const int at = warp * S::ROWS + r * 8 + t4 * 2 + e;
      if (gq == 0) part[at] = make_float2(m[r][e], x);
#pragma unroll
      for (int n = 0; n < S::MT; ++n) *reinterpret_cast<float2*>(os + at * VDIM + S::channel(n, gq)) = make_float2(o[r][n][e], o[r][n][2 + e]);
    }
  __syncthreads();
  constexpr int N = VDIM / 32, ROWS = S::ROWS;
  const long long rows = (long long)a.M * a.H;
  for (int r = warp; r < ROWS && r0 + r < R; r += WARPS) {
    const int i = (r0 + r) / a.rep, h = g * a.rep + (r0 + r) - i * a.rep;
    float top = NONE, sum = 0.f, y[N] = {};
#pragma unroll
    for (int w = 0; w < WARPS; ++w) top = fmaxf(top, part[w * ROWS + r].x);
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
      const float2 x = part[w * ROWS + r];
      const float f = ex2(x.x - top);
      sum = fmaf(x.y, f, sum);
#pragma unroll
      for (int c = 0; c < N; ++c) y[c] = fmaf(os[(w * ROWS + r) * VDIM + lane * N + c], f, y[c]);
    }
    if (a.splits == 1) {
      put_row<DIM, VDIM, KIND>(a, p, i, h, y, sum);
    } else if (a.splits <= CLUSTER) {                              // (in the place of the first warp's part, which this warp alone has read: with all lanes, before one of them writes)
#pragma unroll
      for (int c = 0; c < N; ++c) os[r * VDIM + lane * N + c] = y[c];
      __syncwarp();
      if (lane == 0) part[r] = make_float2(top, sum);
    } else {
      const long long at = blockIdx.x * rows + (long long)(p.row + i) * a.H + h;
#pragma unroll
      for (int c = 0; c < N; ++c) a.ws[at * VDIM + lane * N + c] = y[c];
      if (lane == 0) reinterpret_cast<float2*>(a.ws + a.splits * rows * VDIM)[at] = make_float2(top, sum);
    }
  }
  meet_cluster<DIM, VDIM, KIND, ROWS>(a, p, r0, R, g, os, part);
}

// How a call is cut: rows of a block, blocks of a portion's rows, blocks that share a history
struct Plan {
  int nr, tiles, splits;                                           // nr: eights of rows; 16 and 32 of them on tcgen05
  int spans;                                                       // 4 bits, up to eight rows: blocks that share all histories alike (0: `splits` blocks for each)
};
// Rows of a key head up to which this file's kernel is taken: above 32 a history would be read a second time here, and with bf16 caches the 32 rows' products, in two parts each, take longer than the
// history's bytes where it is long.  us, tcgen05 | here: 58 rows behind 4099 positions, 8 sequences and 8 key heads, e4m3 62 | 73, bf16 65 | 114; 64 rows behind 131003, one sequence, int8 121 | 213, bf16 137 | 366;
// 33 rows behind 280, 64 sequences and 56 key heads, int8 340 | 407, bf16 326 | 541; 17 of them 341 | 225, 322 | 301; 28 behind 1000, 30 sequences and 8 key heads, int8 47 | 41, bf16 51 | 68;
// 32 behind 131003 int8 121 | 122, bf16 138 | 213; 16 behind as many int8 120 | 86, bf16 136 | 102.  4 bits: 32 behind 131003 128 | 99, 32 behind 8000, 16 sequences and 8 key heads, 131 | 103, 31 behind
// 280, 64 sequences and 56 key heads, 347 | 232.
int rows_here(int type, long long span) { return type == LIA_CACHE_BF16 && span > 512 ? 16 : 32; }
long long span_of(int rows, int max_ctx, int window) { return window > 0 && (long long)window + rows < max_ctx ? (long long)window + rows : max_ctx; }
// Histories of four bits: up to eight rows of a key head in equal spans of all histories together, which no block has more of than another, and a second launch that joins; or so many blocks a history,
// and a cluster that joins.  us, spans | splits: a token of 16 requests behind 30001 positions, 16 heads on 8, 111 | 124, of requests behind 21000 to 30001 97 | 116, behind 3000 to 30001 71 | 107; of 32
// behind 8000, 8 heads on 8 (3459 keys a block) 68 | 69; of 64 behind 2000, 32 heads on 8 (1729) 53 | 49; of 16 behind 1901 (411) 20 | 14.
constexpr long long SPAN_KEYS = 3000;                              // of a block, from which on
Plan cut(int nr, long long R, int nseg, int rows, int max_ctx, int G, int window, int type) {
  Plan p{};
  p.nr = nr;
  p.tiles = (int)((R + 8 * p.nr - 1) / (8 * p.nr));
  const long long blocks = (long long)nseg * G * p.tiles, room = (long long)lia_sm_count() * (p.nr >= 16 ? 1 : blocks_an_sm(type, p.nr));
  const long long span = span_of(rows, max_ctx, window);
  const long long least = p.nr >= 16 ? 512 : 256;                   // keys of a block of threads: eight blocks of 64, or four of 16 a warp
  long long s = room / blocks, most = (span + least - 1) / least;
  if (s > most) s = most;
  if (s > MAX_SPLITS) s = MAX_SPLITS;
  p.splits = s < 1 ? 1 : (int)s;
  if (type == LIA_CACHE_INT4 && nr == 1 && blocks * span >= room * SPAN_KEYS) p.spans = (int)(room / G);
  return p;
}
// About how long a plan takes on tcgen05, in us, fitted to 13 measured calls (within a fifth, most of them): a block of threads with up to 128 rows 8 and 0.75 for 64 keys, one with 256 rows 20 and
// 1.2; the first tiles of a portion see fewer keys than the last ones; a second launch 4.
float tc_time(const Plan& p, long long R, int nseg, int rows, int max_ctx, int G, int window) {
  const float tile = 8.f * p.nr, tokens = fminf(rows, rows * tile / R), hidden = window > 0 ? 0.f : rows - tokens, span = window > 0 ? fminf(max_ctx, window + tokens) : max_ctx;
  auto of = [&](bool large, float keys) { return (large ? 20.f : 8.f) + (large ? 1.2f : 0.75f) * fmaxf(keys, 0.f) / (64.f * p.splits); };
  const float longest = of(p.nr == 32, span), last = of(p.nr == 32 && (R - 1) % 256 >= 128, span), shortest = of(p.nr == 32, span - hidden);
  const float mean = ((p.tiles - 1) * 0.5f * (longest + shortest) + last) / p.tiles, rounds = (float)nseg * G * p.tiles * p.splits / lia_sm_count();
  return (rounds <= 1.f ? longest : fmaxf(longest, rounds * mean)) + (p.splits > 1 ? 4.f : 0.f);
}
// Of more than 128 rows tiles of 256 bring keys once instead of twice, tiles of 128 share the SMs out more evenly and leave less of the last one empty.  us, 256 | 128, two portions behind 512
// positions and some, 16 heads on 8, int8: of 200 tokens 29 | 20, 400 34 | 22, 1003 51 | 43, 2000 98 | 105, 4001 258 | 278; of 333 behind 4000 62 | 71; one of 1003 43 | 30.
Plan plan_of(int nseg, int rows, int max_ctx, int H, int G, int window, int type) {
  const long long R = (long long)rows * (H / G);
  auto of = [&](int nr) { return cut(nr, R, nseg, rows, max_ctx, G, window, type); };
  if (R <= rows_here(type, span_of(rows, max_ctx, window))) return of(R > 16 ? 4 : R > 8 ? 2 : 1);
  const Plan one = of(16);
  if (R <= 128) return one;
  const Plan two = of(32);
  return tc_time(two, R, nseg, rows, max_ctx, G, window) <= tc_time(one, R, nseg, rows, max_ctx, G, window) ? two : one;
}
size_t floats_of(const Plan& p, int nseg, int rows, int M, int H, int G, int vdim) {
  if (p.spans > 0) return ((size_t)nseg + p.spans) * G * rows * (H / G) * (vdim + 2);
  return p.splits > (p.nr >= 16 ? 1 : CLUSTER) ? (size_t)p.splits * M * H * (vdim + 2) : 0;
}

template <int DIM, int VDIM, int KIND, int NR> int launch(const TreeArgs& a, int nseg, cudaStream_t stream) {
  using S = Shape<DIM, VDIM, KIND, NR>;
  static bool configured[64] = {};                                 // per device
  int dev = 0;
  LIA_CUDA(cudaGetDevice(&dev));
  if (S::SMEM > 48 * 1024 && (dev >= 64 || !configured[dev])) {
    LIA_CUDA(cudaFuncSetAttribute(tree_attn_kernel<DIM, VDIM, KIND, NR>, cudaFuncAttributeMaxDynamicSharedMemorySize, S::SMEM));
    if (dev < 64) configured[dev] = true;
  }
  const dim3 grid(a.splits, a.tiles * a.G, nseg);
  if (a.splits > 1 && a.splits <= CLUSTER) LIA_CUDA(lia_launch_cluster(a.splits, tree_attn_kernel<DIM, VDIM, KIND, NR>, grid, dim3(THREADS), S::SMEM, stream, a));
  else LIA_CUDA(lia_launch(tree_attn_kernel<DIM, VDIM, KIND, NR>, grid, dim3(THREADS), S::SMEM, stream, a));
  return LIA_OK;
}
template <int DIM, int VDIM, int KIND> int launch_rows(const TreeArgs& a, int nr, int nseg, cudaStream_t stream) {
  int rc;
  if (nr >= 16) rc = lia_tree_attn_tc(&a, KIND, nr * 8, nseg, stream);
  else if constexpr (KIND == LIA_CACHE_INT4) rc = lia_tree_attn_4bit(&a, nr, nseg, stream);
  else rc = nr == 4 ? launch<DIM, VDIM, KIND, 4>(a, nseg, stream) : nr == 2 ? launch<DIM, VDIM, KIND, 2>(a, nseg, stream) : launch<DIM, VDIM, KIND, 1>(a, nseg, stream);
  if (rc == LIA_OK && a.spans == 0 && a.splits > (nr >= 16 ? 1 : CLUSTER)) LIA_CUDA(lia_launch(tree_attn_join_kernel<DIM, VDIM, KIND>, dim3((unsigned)(((long long)a.rows * a.H + 3) / 4), nseg), dim3(128), 0, stream, a));
  return rc;
}
template <int KIND> int launch_dims(const TreeArgs& a, int nr, int nseg, cudaStream_t stream) {
  if (a.k.dim == 128) return a.v.dim == 128 ? launch_rows<128, 128, KIND>(a, nr, nseg, stream) : launch_rows<128, 64, KIND>(a, nr, nseg, stream);
  return a.v.dim == 128 ? launch_rows<64, 128, KIND>(a, nr, nseg, stream) : launch_rows<64, 64, KIND>(a, nr, nseg, stream);
}

}  // namespace

extern "C" size_t lia_tree_attn_workspace_floats(int nseg, int rows, int max_ctx, int M, int H, int G, int dim, int vdim, int window, int type) {
  (void)dim;
  if (nseg <= 0 || rows <= 0 || M <= 0 || G <= 0 || H <= 0 || H % G || vdim <= 0) return 0;
  return floats_of(plan_of(nseg, rows, max_ctx, H, G, window, type), nseg, rows, M, H, G, vdim);
}

extern "C" int lia_tree_attn_plan(int nseg, int rows, int max_ctx, int H, int G, int window, int type) {
  if (nseg <= 0 || rows <= 0 || G <= 0 || H <= 0 || H % G) return 0;
  const Plan p = plan_of(nseg, rows, max_ctx, H, G, window, type);
  return (p.spans > 0 ? 1 << 30 | p.spans << 8 : p.splits << 8) | p.nr;
}

extern "C" int lia_tree_attn(const void* q, long long ldq, const LiaCacheView* kc, const LiaCacheView* vc, const int* segs, int nseg, const long long* mask, int words, const int* depth,
                             const float* temp, void* out, float* ws, size_t ws_floats, int M, int H, int G, int rows, int max_ctx, int window, float scale, float softcap, lia_stream_t stream_) {
  cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_);
  const char* wrong;
  LIA_CHECK_ARG(!(wrong = cache8_wrong(kc, 16)) && !(wrong = cache8_wrong(vc, 16)), "lia_tree_attn: %s", wrong);
  LIA_CHECK_ARG((kc->dim == 64 || kc->dim == 128) && (vc->dim == 64 || vc->dim == 128), "lia_tree_attn: heads have 64 or 128 channels, not %d and %d", kc->dim, vc->dim);
  LIA_CHECK_ARG(kc->type == vc->type && kc->slots == vc->slots && kc->capacity == vc->capacity, "lia_tree_attn: caches of different types or sizes");
  LIA_CHECK_ARG(kc->capacity <= 1 << 29, "lia_tree_attn: more than 2^29 positions");               // (positions, depths and windows are added up in 32 bits)
  LIA_CHECK_ARG(M >= 0 && nseg >= 0 && rows >= 0 && max_ctx >= 0 && G > 0 && H > 0 && H % G == 0, "lia_tree_attn: bad sizes");
  LIA_CHECK_ARG(!(softcap > MOST_SOFTCAP), "lia_tree_attn: a soft cap of %g is more than %g", softcap, MOST_SOFTCAP);
  if (M == 0 || nseg == 0 || rows == 0) return LIA_OK;
  LIA_CHECK_ARG(q && segs && out && (mask == nullptr || words > 0), "lia_tree_attn: null pointer");
  LIA_CHECK_ARG(ldq >= (long long)H * kc->dim && ldq % 4 == 0 && reinterpret_cast<uintptr_t>(q) % 8 == 0 && reinterpret_cast<uintptr_t>(out) % 8 == 0, "lia_tree_attn: queries and outputs have to be whole 8-byte vectors");
  LIA_CHECK_ARG(mask == nullptr || rows <= 64 * words, "lia_tree_attn: %d words of mask do not hold %d tokens", words, rows);
  const Plan plan = plan_of(nseg, rows, max_ctx, H, G, window, kc->type);
  LIA_CHECK_ARG(nseg <= 65535 && (long long)plan.tiles * G <= 65535, "lia_tree_attn: too many portions, or rows of one");
  LIA_CHECK_ARG(floats_of(plan, nseg, rows, M, H, G, vc->dim) == 0 || (ws && ws_floats >= floats_of(plan, nseg, rows, M, H, G, vc->dim) && reinterpret_cast<uintptr_t>(ws) % 16 == 0), "lia_tree_attn: needs a workspace of %zu floats",
                floats_of(plan, nseg, rows, M, H, G, vc->dim));
  const TreeArgs a{reinterpret_cast<const bf16*>(q), ldq, cache8(kc), cache8(vc), segs, reinterpret_cast<const unsigned long long*>(mask), words, depth, temp,
                   reinterpret_cast<bf16*>(out), ws, M, H, G, H / G, rows, window > 0 ? window : 1 << 30, plan.splits, plan.tiles, scale, softcap, nseg, plan.spans};
  switch (kc->type) {
    case LIA_CACHE_BF16: return launch_dims<LIA_CACHE_BF16>(a, plan.nr, nseg, stream);
    case LIA_CACHE_INT8: return launch_dims<LIA_CACHE_INT8>(a, plan.nr, nseg, stream);
    case LIA_CACHE_INT4: return launch_dims<LIA_CACHE_INT4>(a, plan.nr, nseg, stream);
    default: return launch_dims<LIA_CACHE_E4M3>(a, plan.nr, nseg, stream);
  }
}
