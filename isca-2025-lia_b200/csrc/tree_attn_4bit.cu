// Attention of drafted or decoded tokens over caches of 4 bits, for up to 32 rows of a key head (tree_attn.cu has the formulas and the plan; more rows: tree_attn_sm100.cu).
//
//   s_ij = cap tanh(temp_h scale sum_g ks_jg (q_ig . k_jg) / cap),   o_ig = sum_j p_ij vs_jg v_jg / sum_j p_ij,   g: groups of 32 channels
//
// As over 8 bits the keys are the products' rows and the queries their columns, and a warp takes 16 keys at a time.  What is different: half the bytes leave half the time, so that instructions count.
//   * Keys, values and scales come to shared memory by cp.async, DEPTH blocks of a warp ahead, and from there as the products want them.
//   * A key's codes are code + 8 = u in 0 .. 15: four bits in the lowest ten of an fp16 number are the subnormal number u 2^-24 (or 16 u 2^-24, whose query is divided by 16), so that one instruction
//     makes two operands.  The sums begin with -8 (the queries' sum) instead of 0.  With more than eight rows the 2^10 and the offset are subtracted from 1024 + u instead, as they are of values with
//     more than two.
//   * A value's group scale multiplies its weight, relative to the value's largest scale, which goes into the exponent (tree_attn.cu).
//   * One or two rows (PACKED; a decoded token of up to two query heads): the eight columns are four quarters of the channels times two rows.  A column's query is nothing but in its quarter, whose
//     group is one, so that a lane has one scale a key instead of four, and a weight goes into the second product once, not once a group.  A word of codes has four channels of two groups, and is taken as
//     it is: what belongs together along the products' sum are the same channel of two groups, of which a column's query or weight is that of its own group, and nothing for the other.  Values' codes are
//     subnormal numbers too: the sums of 16 keys begin with -8 (their weights' sum), and are added to what was before (over all keys that would be large beside what they average out to; of 16 it leaves
//     2^-13 of a weight times its value's scale at most, where a weight's own rounding leaves 2^-11 of a weight times its value).
//
// 16 tokens behind 21000 to 30001 positions, 16 heads on 8 (475 MB): 98 us, 4.9 TB/s, 74 % of the copy rate, the second launch among them; with the 8-bit kernel's structure 207.  What bounds it:
// instructions, some 290 a warp for 16 keys (488 at first; 342 with values' codes less 1032 instead of subnormal, 110 us), half of them on the integer pipe (51 % busy, issue slots 62 %), and memory next;
// five or six blocks an SM change nothing (99.5, 100), nor do shorter spans (twice as many 112).
// More rows of a key head: the same histories with 4 or 8 rows 123 us, 16 rows 208, 32 rows 342 (issue slots 66, 62 and 50 % busy, 3.2, 2.5 and 1.7 warps a scheduler): scores and weights by rows times groups.
#include "mma.cuh"
#include "tree_attn.cuh"

namespace {

constexpr int DEPTH = 4;                                           // blocks of 16 keys of a warp on their way

// c = a b + d
__device__ __forceinline__ void mma_f16_from(float* c, const uint32_t* a, uint32_t b0, uint32_t b1, const float* d) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
               : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(d[0]), "f"(d[1]), "f"(d[2]), "f"(d[3]));
}
// as int4x2, but u 2^-24 (j = 0, 2) and 16 u 2^-24 (1, 3)
__device__ __forceinline__ void small4x2(uint32_t w, uint32_t (&r)[4]) {
  r[0] = w & 0x000f000fu;
  r[1] = w & 0x00f000f0u;
  const uint32_t x = w >> 8;
  r[2] = x & 0x000f000fu;
  r[3] = x & 0x00f000f0u;
}
__device__ __forceinline__ float rcp(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
template <int BYTES> __device__ __forceinline__ void cp_async_small(uint32_t dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(dst), "l"(src), "n"(BYTES) : "memory");
}
__device__ __forceinline__ uint32_t lds32(uint32_t at) {
  uint32_t v;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(at) : "memory");
  return v;
}
__device__ __forceinline__ uint2 lds64(uint32_t at) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(at) : "memory");
  return v;
}
__device__ __forceinline__ uint4 lds128(uint32_t at) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at) : "memory");
  return v;
}
__device__ __forceinline__ float lds_bf16(uint32_t at) {
  uint16_t v;
  asm volatile("ld.shared.u16 %0, [%1];" : "=h"(v) : "r"(at) : "memory");
  return __uint_as_float((uint32_t)v << 16);
}

template <int DIM, int VDIM, int NR> struct Four {
  static constexpr int KG = DIM / GROUP4, VG = VDIM / GROUP4, STEPS = DIM / 16, MT = VDIM / 16, ROWS = 8 * NR;
  static constexpr int KROW = DIM / 2, VROW = VDIM / 2;            // bytes of a key, of a value
  static constexpr int KS_AT = 16 * (KROW + VROW), VS_AT = KS_AT + 16 * KG * 2, STAGE = VS_AT + 16 * VG * 2;
  static constexpr int RING = WARPS * DEPTH * STAGE, Q_BYTES = NR * STEPS * 32 * 8, O_BYTES = WARPS * ROWS * VDIM * 4;
  static constexpr int BIG = Q_BYTES + RING > O_BYTES ? Q_BYTES + RING : O_BYTES;
  static constexpr int SMEM = BIG + ROWS * 4 + WARPS * ROWS * 8 + ROWS * KG * 4;
};
constexpr float LIFT = 7.f;                                        // a weight of the maximum is 2^LIFT, one that is just not outgrown 2^15 in fp16

// of value row i (the product's number i along the keys) where its 16-byte chunk c lies: rows whose lanes read at the same time (2 t4 and 8 + 2 t4 for t4 = 0 .. 3) in different banks
template <int VROW> __device__ __forceinline__ int value_at(int i, int c) {
  const int r = (i >> 1) | (i & 1) << 3;
  return VROW == 64 ? r * 64 + ((c ^ (r & 2)) << 4) : r * VROW + (c << 4);
}

// What a block of threads works on: rows r0 .. of a portion and a key head, blocks b0 .. b1 - 1 of 16 keys from position lo on
struct Piece {
  int g, r0, lo, hi, all_lo, all_hi, b0, b1;
};
template <int DIM, int VDIM, int NR> struct Shared {
  using S = Four<DIM, VDIM, NR>;
  float* row_f;                                                    // [ROWS] what a row's products with keys are multiplied by
  float2* part;                                                    // [WARPS][ROWS] maximum, sum
  float* row_q;                                                    // [ROWS][KG] -8 2^-24 times the sum of a group's queries
  uint2* qs;                                                       // [NR][STEPS][32]
  float* os;                                                       // [WARPS][ROWS][VDIM] weighted values, where queries and rings were
  __device__ __forceinline__ explicit Shared(uint4* smem) {
    row_f = reinterpret_cast<float*>(reinterpret_cast<uint8_t*>(smem) + S::BIG);
    part = reinterpret_cast<float2*>(row_f + S::ROWS);
    row_q = reinterpret_cast<float*>(part + WARPS * S::ROWS);
    qs = reinterpret_cast<uint2*>(smem);
    os = reinterpret_cast<float*>(smem);
  }
};

// leaves the warps' sums in sh.os and sh.part, behind a barrier
template <int DIM, int VDIM, int NR, bool PACKED> __device__ __forceinline__ void run_piece(const TreeArgs& a, const Portion& p, const Piece& pc, const Shared<DIM, VDIM, NR>& sh) {
  using S = Four<DIM, VDIM, NR>;
  constexpr bool SMALL = NR == 1;                                  // keys' codes as subnormal numbers
  static_assert(!PACKED || NR == 1, "one or two rows");
  const int warp = __shfl_sync(0xffffffffu, (int)threadIdx.x >> 5, 0), lane = threadIdx.x & 31, gq = lane >> 2, t4 = lane & 3;   // (known to be the same in all lanes)
  const int g = pc.g, r0 = pc.r0, lo = pc.lo, hi = pc.hi, all_lo = pc.all_lo, all_hi = pc.all_hi, b0 = pc.b0, b1 = pc.b1, R = p.n * a.rep;
  float* row_f = sh.row_f;
  float2* part = sh.part;
  float* row_q = sh.row_q;
  uint2* qs = sh.qs;

  // ---- the ring: a lane brings 16-byte chunks of keys and values lane / CH (and 8 more, where a row has four chunks), lanes 0 .. 15 a key's scales, the others a value's
  const uint32_t ring = smem_u32(sh.qs) + S::Q_BYTES + warp * DEPTH * S::STAGE;
  constexpr int KCH = S::KROW / 16, VCH = S::VROW / 16, KN = 16 * KCH / 32, VN = 16 * VCH / 32;  // chunks of a row; copies of a lane
  const int sgroups = lane < 16 ? S::KG : S::VG, start = lo + (b0 + warp) * 16;                // the warp's first block
  const uint8_t *kp = a.k.at(p.slot, start, g) + lane / KCH * a.k.pos + lane % KCH * 16, *vp = a.v.at(p.slot, start, g) + lane / VCH * a.v.pos + lane % VCH * 16;
  const bf16* sp = (lane < 16 ? a.k.scale4_at(p.slot, g) : a.v.scale4_at(p.slot, g)) + (long long)(start + (lane & 15)) * sgroups;
  const long long k_step = WARPS * 16 * a.k.pos, v_step = WARPS * 16 * a.v.pos;
  const uint32_t k_to = lane * 16, s_to = lane < 16 ? S::KS_AT + lane * S::KG * 2 : S::VS_AT + (lane - 16) * S::VG * 2;
  auto bring = [&](int b, int stage) {
    if (b < b1) {
      const uint32_t at = ring + stage * S::STAGE;
      const int last = hi - 1 - (lo + b * 16);                     // of the block: keys behind it are that one again
      const bf16* src = sp;
      if (last >= 15) {
#pragma unroll
        for (int n = 0; n < KN; ++n) cp_async16(at + k_to + n * 512, kp + n * 8 * a.k.pos, 16);
#pragma unroll
        for (int n = 0; n < VN; ++n) cp_async16(at + 16 * S::KROW + value_at<S::VROW>(lane / VCH + n * 8, lane % VCH), vp + n * 8 * a.v.pos, 16);
      } else {
#pragma unroll
        for (int n = 0; n < KN; ++n) cp_async16(at + k_to + n * 512, kp + (long long)(min(lane / KCH + n * 8, last) - lane / KCH) * a.k.pos, 16);
#pragma unroll
        for (int n = 0; n < VN; ++n) {
          const int i = lane / VCH + n * 8;
          cp_async16(at + 16 * S::KROW + value_at<S::VROW>(i, lane % VCH), vp + (long long)(min(i, last) - lane / VCH) * a.v.pos, 16);
        }
        src += (min(lane & 15, last) - (lane & 15)) * sgroups;
      }
      if constexpr (S::KG == S::VG) {
        cp_async_small<S::KG * 2>(at + s_to, src);
      } else {
        if (lane < 16) cp_async_small<S::KG * 2>(at + s_to, src);
        else cp_async_small<S::VG * 2>(at + s_to, src);
      }
      kp += k_step;
      vp += v_step;
      sp += WARPS * 16 * sgroups;
    }
    cp_async_commit();
  };
#pragma unroll
  for (int d = 0; d < DEPTH; ++d) bring(b0 + warp + d * WARPS, d); // (on their way while the queries are brought)

  // ---- queries: rows (token, head) in the order of the products' operands
  constexpr int MINE = S::ROWS / WARPS;                            // rows of a warp, asked for together
  uint2 asked[MINE];
  float temps[MINE];
#pragma unroll
  for (int x = 0; x < MINE; ++x) {
    const int r = warp + x * WARPS, i = (r0 + r) / a.rep, h = g * a.rep + (r0 + r) - i * a.rep;
    asked[x] = r0 + r < R && lane < DIM / 4 ? *reinterpret_cast<const uint2*>(a.q + (p.row + i) * a.ldq + h * DIM + lane * 4) : make_uint2(0u, 0u);
    temps[x] = a.temp != nullptr && r0 + r < R ? a.temp[h] : 1.f;
  }
#pragma unroll
  for (int x = 0; x < MINE; ++x) {
    const int r = warp + x * WARPS;
    const uint2 u = asked[x];
    float f = a.scale * temps[x] * (a.softcap > 0.f ? 1.f : LOG2E);
    const uint32_t top = max(max((u.x & 0x7fffu), (u.x >> 16) & 0x7fffu), max((u.y & 0x7fffu), (u.y >> 16) & 0x7fffu));
    const Down down = down_of(__reduce_max_sync(0xffffffffu, top));
    float y[4];
    unpack_bf16x2(u.x, y[0], y[1]);
    unpack_bf16x2(u.y, y[2], y[3]);
    constexpr float ODD = SMALL ? 0.0625f : 1.f;                   // channels 1, 3, 5, 7 of every eight go with 16 u
    uint2 w = make_uint2(pack_f16x2(y[0] * down.by, y[1] * down.by * ODD), pack_f16x2(y[2] * down.by, y[3] * down.by * ODD));
    f *= down.back;
    w = in_code_order(w);                                          // of eight channels an even lane has 0 4 1 5, an odd one 2 6 3 7: their operands of two steps
    if constexpr (SMALL) {
      f *= 0x1p24f;
      const float2 c0 = __half22float2(*reinterpret_cast<const __half2*>(&w.x)), c1 = __half22float2(*reinterpret_cast<const __half2*>(&w.y));
      float sum = (c0.x + c0.y) + 16.f * (c1.x + c1.y);
      sum += __shfl_xor_sync(0xffffffffu, sum, 2);
      sum += __shfl_xor_sync(0xffffffffu, sum, 4);
      if (!PACKED || DIM == 128) sum += __shfl_xor_sync(0xffffffffu, sum, 1);                  // (a quarter is a group's two steps, or one)
      const int gr = lane >> 3, step = lane & 1;
      if constexpr (PACKED) {
        if (r < 2 && (lane & 6) == 0 && lane < DIM / 4) row_q[r * 4 + (DIM == 128 ? gr : gr * 2 + step)] = -8.f * 0x1p-24f * sum;
      } else if ((lane & 7) == 0 && lane < DIM / 4) {
        row_q[r * S::KG + gr] = -8.f * 0x1p-24f * sum;
      }
    }
    if (lane < DIM / 4) {
      const int c = lane * 4, t = (c >> 3) & 3, step = (c >> 5) * 2 + ((c >> 2) & 1);
      qs[((r >> 3) * S::STEPS + step) * 32 + (r & 7) * 4 + t] = w;
    }
    if (lane == 0) row_f[r] = f;
  }
  __syncthreads();
  uint2 qa[NR == 1 ? S::STEPS : 1];                                // few rows' queries stay in registers, the others' in shared memory
  constexpr int PER = 4 / S::KG, VPER = 4 / S::VG;                 // (PACKED) quarters of a group of keys' and of values' channels: 1 or 2
  uint32_t lower[2], upper[2];                                     // (PACKED) where of a word of two groups' weights those of a column's group go
  if constexpr (PACKED) {                                          // column gq: row gq & 1, in quarter gq >> 1.  A key's word has the same four channels of two groups: a step has two of them, of either group
    const int quarter = gq >> 1, group = quarter / PER, vgroup = quarter / VPER;
#pragma unroll
    for (int w = 0; w < S::STEPS / 2; ++w)
#pragma unroll
      for (int st = 0; st < 2; ++st) {
        const uint2 u = qs[(group * 2 + st) * 32 + (gq & 1) * 4 + t4];
        const int pairs = S::KG / 2, four = w / pairs;             // the group's four 2 t4 or 2 t4 + 1
        const bool mine = group / 2 == w % pairs && (PER == 1 || (quarter & 1) == st);
        const uint32_t to = !mine ? 0x4444u : four == 0 ? (group & 1 ? 0x1044u : 0x4410u) : (group & 1 ? 0x3244u : 0x4432u);
        qa[w * 2 + st] = make_uint2(__byte_perm(u.x, 0u, to), __byte_perm(u.y, 0u, to));
      }
#pragma unroll
    for (int h = 0; h < S::VG / 2; ++h) {
      const bool mine = vgroup / 2 == h && quarter % VPER == 0;
      lower[h] = !mine ? 0x4444u : vgroup & 1 ? 0x1044u : 0x4410u;
      upper[h] = !mine ? 0x4444u : vgroup & 1 ? 0x3244u : 0x4432u;
    }
  } else if constexpr (NR == 1) {
#pragma unroll
    for (int s = 0; s < S::STEPS; ++s) qa[s] = qs[s * 32 + lane];
  }

  // of the lane's columns: rows 2 t4 and 2 t4 + 1 of every eight, or (PACKED) rows 0 and 1 in quarter t4
  float rf[NR][2], m[NR][2], l[NR][2];
#pragma unroll
  for (int r = 0; r < NR; ++r)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      rf[r][e] = row_f[PACKED ? e : r * 8 + t4 * 2 + e];
      m[r][e] = NONE;
      l[r][e] = 0.f;
    }
  float from[PACKED ? 1 : S::KG][SMALL ? 2 : 1];
  if constexpr (SMALL) {
#pragma unroll
    for (int gr = 0; gr < (PACKED ? 1 : S::KG); ++gr)
#pragma unroll
      for (int e = 0; e < 2; ++e) from[gr][e] = PACKED ? row_q[e * 4 + t4] : row_q[(t4 * 2 + e) * S::KG + gr];
  }
  constexpr int MT = PACKED ? 2 : S::MT;
  float o[NR][MT][4];                                              // [..][0]: a lane's first channel of a pair and row 2 t4, [1]: row 2 t4 + 1, [2], [3]: its second channel (PACKED: of group t4 / VPER)
#pragma unroll
  for (int r = 0; r < NR; ++r)
#pragma unroll
    for (int n = 0; n < MT; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[r][n][e] = 0.f;

  const float two_by_cap = a.softcap > 0.f ? 2.f * LOG2E / a.softcap : 0.f;
  const uint32_t k_from = gq * S::KROW + t4 * (S::KROW / 4), v_from = 16 * S::KROW + (gq * (S::VROW / 8) & 15);
  int stage = 0;
#pragma unroll 1
  for (int b = b0 + warp; b < b1; b += WARPS) {
    cp_async_wait<DEPTH - 1>();
    __syncwarp();
    const uint32_t at = ring + stage * S::STAGE;
    // ---- products of 16 keys and all rows: s[r][0], [1]: key gq and the lane's two columns; [2], [3]: key gq + 8
    uint32_t kr[2][S::KROW / 16];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      if constexpr (DIM == 128) *reinterpret_cast<uint4*>(kr[j]) = lds128(at + k_from + j * 8 * S::KROW);
      else *reinterpret_cast<uint2*>(kr[j]) = lds64(at + k_from + j * 8 * S::KROW);
    }
    float s[NR][4];
    auto codes_of = [&](int j, int gr) { return __byte_perm(kr[j][gr >> 1], kr[j][S::KG / 2 + (gr >> 1)], gr & 1 ? 0x7632 : 0x5410); };
    if constexpr (PACKED) {
      float even[4] = {from[0][0], from[0][1], from[0][0], from[0][1]}, odd[4] = {};
#pragma unroll
      for (int w = 0; w < S::STEPS / 2; ++w) {
        uint32_t codes[2][4];
#pragma unroll
        for (int j = 0; j < 2; ++j) small4x2(kr[j][w], codes[j]);
#pragma unroll
        for (int st = 0; st < 2; ++st) {
          const uint32_t ka[4] = {codes[0][2 * st], codes[1][2 * st], codes[0][2 * st + 1], codes[1][2 * st + 1]};
          mma_f16(st == 0 ? even : odd, ka, qa[w * 2 + st].x, qa[w * 2 + st].y);
        }
      }
      float kg[2];
#pragma unroll
      for (int j = 0; j < 2; ++j) kg[j] = lds_bf16(at + S::KS_AT + ((gq + j * 8) * S::KG + t4 / PER) * 2);
#pragma unroll
      for (int e = 0; e < 4; ++e) s[0][e] = (even[e] + odd[e]) * kg[e >> 1];
#pragma unroll
      for (int x = 1; x < 4; x <<= 1)                              // the quarters' lanes together
#pragma unroll
        for (int e = 0; e < 4; ++e) s[0][e] += __shfl_xor_sync(0xffffffffu, s[0][e], x);
    } else {
      uint32_t ks4[2][S::KG / 2];
      float kg[2][S::KG];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        if constexpr (S::KG == 4) *reinterpret_cast<uint2*>(ks4[j]) = lds64(at + S::KS_AT + (gq + j * 8) * 8);
        else ks4[j][0] = lds32(at + S::KS_AT + (gq + j * 8) * 4);
        scales4_of<S::KG>(ks4[j], kg[j]);
      }
#pragma unroll
      for (int r = 0; r < NR; ++r)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[r][e] = 0.f;
#pragma unroll
      for (int gr = 0; gr < S::KG; ++gr) {                         // group by group, whose sums are multiplied by their scales
        uint32_t codes[2][4];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          if constexpr (SMALL) small4x2(codes_of(j, gr), codes[j]);
          else int4x2(codes_of(j, gr), codes[j]);
        }
#pragma unroll
        for (int r = 0; r < NR; ++r) {
          float sum[4] = {};
#pragma unroll
          for (int st = 0; st < 2; ++st) {
            const uint32_t ka[4] = {codes[0][2 * st], codes[1][2 * st], codes[0][2 * st + 1], codes[1][2 * st + 1]};
            uint2 q;
            if constexpr (NR == 1) q = qa[gr * 2 + st];
            else q = qs[(r * S::STEPS + gr * 2 + st) * 32 + lane];
            if (SMALL && st == 0) {
              const float start[4] = {from[gr][0], from[gr][SMALL], from[gr][0], from[gr][SMALL]};
              mma_f16_from(sum, ka, q.x, q.y, start);
            } else {
              mma_f16(sum, ka, q.x, q.y);
            }
          }
#pragma unroll
          for (int e = 0; e < 4; ++e) s[r][e] = fmaf(sum[e], kg[e >> 1][gr], s[r][e]);
        }
      }
    }
    // ---- values' scales: the largest goes into the exponent, the others relative to it onto the weights
    constexpr int VS = PACKED ? 1 : S::VG;
    float lv[2], rv[2], ratio[2][VS];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const uint32_t from_at = at + S::VS_AT + (gq + j * 8) * S::VG * 2;
      uint32_t vs4[S::VG / 2];
      if constexpr (S::VG == 4) *reinterpret_cast<uint2*>(vs4) = lds64(from_at);
      else vs4[0] = lds32(from_at);
      // (numbers of 0 and more compare as whole numbers, NaN above them)
      const uint32_t two = S::VG == 4 ? __vmaxu2(vs4[0], vs4[S::VG / 2 - 1]) : vs4[0];
      const float y = max_nan(__uint_as_float(max(two << 16, two & 0xffff0000u)), LEAST_SCALE);
      lv[j] = lg2(y);
      rv[j] = rcp(y);
      if constexpr (PACKED) {
        ratio[j][0] = lds_bf16(from_at + t4 / VPER * 2) * rv[j];
      } else {
        scales4_of<S::VG>(vs4, ratio[j]);
#pragma unroll
        for (int gr = 0; gr < S::VG; ++gr) ratio[j][gr] *= rv[j];
      }
    }
    // ---- scores, as powers of two and with the values' scales
    const int key0 = lo + b * 16;
    if (a.softcap > 0.f) {
#pragma unroll
      for (int r = 0; r < NR; ++r)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[r][e] = fmaf(capped(s[r][e] * rf[r][e & 1], a.softcap, two_by_cap), LOG2E, lv[e >> 1]);
    } else {
#pragma unroll
      for (int r = 0; r < NR; ++r)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[r][e] = fmaf(s[r][e], rf[r][e & 1], lv[e >> 1]);
    }
    if (key0 < all_lo || key0 + 16 > all_hi) {
#pragma unroll
      for (int r = 0; r < NR; ++r)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int i = min((r0 + (PACKED ? e : r * 8 + t4 * 2 + e)) / a.rep, p.n - 1), d = depth_of(a, p, i);
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
      for (int e = 0; e < 2; ++e) grown |= fmaxf(s[r][e], s[r][2 + e]) - m[r][e] > SLACK + LIFT;
    if (__any_sync(0xffffffffu, grown)) {
#pragma unroll
      for (int r = 0; r < NR; ++r)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float top = fmaxf(s[r][e], s[r][2 + e]);
#pragma unroll
          for (int x = 4; x < 32; x <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
          const bool up = top - m[r][e] > SLACK + LIFT;
          const float keep = up ? ex2(m[r][e] - (top - LIFT)) : 1.f;
          if (up) m[r][e] = top - LIFT;
          l[r][e] *= keep;
#pragma unroll
          for (int n = 0; n < MT; ++n) {
            o[r][n][e] *= keep;
            o[r][n][2 + e] *= keep;
          }
        }
    }
    // ---- weights, turned into the products' other operand
    uint32_t pb[VS][NR][2];
#pragma unroll
    for (int r = 0; r < NR; ++r) {
      float w[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        w[e] = ex2(s[r][e] - m[r][e & 1]);
        l[r][e & 1] = fmaf(w[e], rv[e >> 1], l[r][e & 1]);
      }
#pragma unroll
      for (int gr = 0; gr < VS; ++gr)
#pragma unroll
        for (int j = 0; j < 2; ++j) pb[gr][r][j] = transposed(pack_f16x2(w[2 * j] * ratio[j][gr], w[2 * j + 1] * ratio[j][gr]));
    }
    // ---- weighted values
    uint32_t vr[4][S::VG / 2];                                     // of keys 2 t4, 2 t4 + 1, 8 + 2 t4, 9 + 2 t4: four channels of every group
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const uint32_t from_at = at + v_from + value_at<S::VROW>((c >> 1) * 8 + t4 * 2 + (c & 1), gq * (S::VROW / 8) >> 4);
      if constexpr (VDIM == 128) *reinterpret_cast<uint2*>(vr[c]) = lds64(from_at);
      else vr[c][0] = lds32(from_at);
    }
    __syncwarp();                                                  // the stage has been read
    bring(b + DEPTH * WARPS, stage);
    stage = stage + 1 == DEPTH ? 0 : stage + 1;
    if constexpr (PACKED) {                                        // 16 keys' sums begin with -8 (the weights' sum): of 16 keys that is no more than the products are
      float sum[2][4] = {};
      constexpr uint32_t OFFSET[4] = {0x80088008u, 0x80808080u, 0x80088008u, 0x80808080u};     // -8 2^-24, and 16 times that
      mma_f16(sum[0], OFFSET, pb[0][0][0], pb[0][0][1]);
#pragma unroll
      for (int e = 0; e < 4; ++e) sum[1][e] = sum[0][e];
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int h = 0; h < S::VG / 2; ++h) {
          uint32_t codes[2][4];                                    // of keys 8 j + 2 t4 and the next one: four channels of two groups
#pragma unroll
          for (int c = 0; c < 2; ++c) small4x2(vr[2 * j + c][h], codes[c]);
          const uint32_t lo16 = __byte_perm(pb[0][0][j], 0u, lower[h]), hi16 = __byte_perm(pb[0][0][j], 0u, upper[h]);
#pragma unroll
          for (int n = 0; n < 2; ++n) {
            const uint32_t v4[4] = {codes[0][2 * n], codes[0][2 * n + 1], codes[1][2 * n], codes[1][2 * n + 1]};
            mma_f16(sum[n], v4, lo16, hi16);
          }
        }
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[0][n][e] += sum[n][e];
    } else {
#pragma unroll
      for (int gr = 0; gr < S::VG; ++gr) {
        uint32_t va[2][4];                                           // a lane's four channels of the group, of keys 2 t4 and 2 t4 + 1, and of those 8 on
#pragma unroll
        for (int c = 0; c < 2; ++c) int4x2(__byte_perm(vr[2 * c][gr >> 1], vr[2 * c + 1][gr >> 1], gr & 1 ? 0x7632 : 0x5410), va[c]);
#pragma unroll
        for (int c = 0; c < 4; c += 2) {
          const uint32_t v4[4] = {va[0][c], va[0][c + 1], va[1][c], va[1][c + 1]};
#pragma unroll
          for (int r = 0; r < NR; ++r) mma_f16(o[r][gr * 2 + (c >> 1)], v4, pb[gr][r][0], pb[gr][r][1]);
        }
      }
    }
  }
  cp_async_wait<0>();

  // ---- the warps' parts meet in shared memory
  __syncthreads();                                                 // (queries and rings have been read)
  float* os = sh.os;
#pragma unroll
  for (int r = 0; r < NR; ++r)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      float x = l[r][e];
#pragma unroll
      for (int d = 4; d < 32; d <<= 1) x += __shfl_xor_sync(0xffffffffu, x, d);
      const int at = warp * S::ROWS + (PACKED ? e : r * 8 + t4 * 2 + e);
      if (gq == 0 && (!PACKED || t4 == 0)) part[at] = make_float2(m[r][e], x);
      if constexpr (PACKED) {
        if (t4 % VPER == 0)
          *reinterpret_cast<float4*>(os + at * VDIM + t4 / VPER * GROUP4 + gq * 4) = make_float4(o[0][0][e] * 0x1p24f, o[0][0][2 + e] * 0x1p20f, o[0][1][e] * 0x1p24f, o[0][1][2 + e] * 0x1p20f);
      } else {
#pragma unroll
        for (int n = 0; n < S::MT; ++n)
          *reinterpret_cast<float2*>(os + at * VDIM + (n >> 1) * GROUP4 + gq * 4 + (n & 1) * 2) = make_float2(o[r][n][e], o[r][n][2 + e]);
      }
    }
  __syncthreads();
}

template <int DIM, int VDIM, int NR, bool PACKED>
__global__ void __launch_bounds__(THREADS, tree_attn4_blocks(NR)) tree_attn4_kernel(const __grid_constant__ TreeArgs a) {
  using S = Four<DIM, VDIM, NR>;
  extern __shared__ uint4 smem[];
  const Shared<DIM, VDIM, NR> sh(smem);
  pdl_launch_dependents();
  pdl_wait();
  const Portion p = portion_of(a, blockIdx.z);
  if (!p.held) {
    if (a.splits <= CLUSTER && blockIdx.x == 0 && blockIdx.y == 0) nan_rows<VDIM>(a, p);
    return;
  }
  const int lane = threadIdx.x & 31;
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
  run_piece<DIM, VDIM, NR, PACKED>(a, p, Piece{g, r0, lo, hi, all_lo, all_hi, b0, b1}, sh);
  // ---- the warps' parts of a row to its output, to shared memory for the cluster, or to the workspace
  constexpr int N = VDIM / 32, ROWS = S::ROWS, KIND = LIA_CACHE_INT4;
  const int warp = __shfl_sync(0xffffffffu, (int)threadIdx.x >> 5, 0);
  float* os = sh.os;
  float2* part = sh.part;
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

// ---- All histories as one list of units of 64 keys (16 for each warp), of which every block of a key head has the same number, whatever the histories' lengths: its span may end one history and begin
// others.  (The heads' blocks of the same span are neighbours: they bring the same positions at the same time, and with them whole lines of memory.)  Span c of head g leaves what it has of portion z in
// slot (z + c) G + g of the workspace, which no other pair (z, c) has, and a second launch joins.
__device__ __forceinline__ int units_of(const TreeArgs& a, int z, int& lo) {
  const Portion p = portion_of(a, z);
  lo = p.held && p.n > 0 ? first_key(a, p, 0) : 0;                 // (of the least depth there can be)
  return p.held && p.n > 0 ? (p.p0 + p.n - lo + WARPS * 16 - 1) / (WARPS * 16) : 0;
}
// by a warp: the portion that unit `u` of the list lies in (a.nseg: behind all of them), how many units come before its first, and how many its history has; u < 0: all units together in `before`
struct Place {
  int z, units;
  long long before;
};
__device__ __forceinline__ Place place_in_list(const TreeArgs& a, long long u) {
  const int lane = threadIdx.x & 31;
  long long before = 0;
  for (int z0 = 0; z0 < a.nseg; z0 += 32) {
    int lo;
    const int mine = z0 + lane < a.nseg ? units_of(a, z0 + lane, lo) : 0;
    long long sum = mine;                                          // up to and with this lane's portion
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long x = __shfl_up_sync(0xffffffffu, sum, o);
      if (lane >= o) sum += x;
    }
    const unsigned behind = u < 0 ? 0u : __ballot_sync(0xffffffffu, before + sum > u);
    if (behind) {
      const int l = __ffs(behind) - 1, n = __shfl_sync(0xffffffffu, mine, l);
      return {z0 + l, n, before + __shfl_sync(0xffffffffu, sum, l) - n};
    }
    before += __shfl_sync(0xffffffffu, sum, 31);
  }
  return {a.nseg, 0, before};
}

template <int DIM, int VDIM, bool PACKED> __global__ void __launch_bounds__(THREADS, tree_attn4_blocks(1)) tree_attn4_spans_kernel(const __grid_constant__ TreeArgs a) {
  using S = Four<DIM, VDIM, 1>;
  constexpr int N = VDIM / 32;
  extern __shared__ uint4 smem[];
  const Shared<DIM, VDIM, 1> sh(smem);
  pdl_launch_dependents();
  pdl_wait();
  const int warp = __shfl_sync(0xffffffffu, (int)threadIdx.x >> 5, 0), lane = threadIdx.x & 31, most = a.rows * a.rep;
  const long long total = place_in_list(a, -1).before, blocks = min((long long)a.spans, total);       // (no block without a unit)
  const int span = blockIdx.x / a.G, g = blockIdx.x - span * a.G;
  if (span >= blocks) return;
  const long long end = total * (span + 1) / blocks;
  long long u = total * span / blocks;
  while (u < end) {
    const Place at = place_in_list(a, u);
    const int z = __shfl_sync(0xffffffffu, at.z, 0), units = __shfl_sync(0xffffffffu, at.units, 0), from = (int)(u - at.before), to = (int)min((long long)units, from + (end - u));
    const Portion p = portion_of(a, z);
    int lo;
    units_of(a, z, lo);
    {
      const int hi = p.p0 + p.n, last = p.n - 1;
      int far = last;
      if (a.depth != nullptr && a.window < 1 << 30) {
        far = lane <= last ? depth_of(a, p, min(lane, last)) : 0;  // (eight tokens at most)
        far = __reduce_max_sync(0xffffffffu, far);
      }
      const int nb = (hi - lo + 15) >> 4;
      run_piece<DIM, VDIM, 1, PACKED>(a, p, Piece{g, 0, lo, hi, first_key(a, p, far), min(hi, a.mask != nullptr ? p.p0 : p.p0 + 1), from * WARPS, min(nb, to * WARPS)}, sh);
      // the warps' sums together, into the slot
      const long long slot = (long long)(z + span) * a.G + g, slots = (long long)(a.nseg + a.spans) * a.G;
      for (int r = warp; r < p.n * a.rep; r += WARPS) {
        float top = NONE, sum = 0.f, y[N] = {};
#pragma unroll
        for (int w = 0; w < WARPS; ++w) top = fmaxf(top, sh.part[w * S::ROWS + r].x);
#pragma unroll
        for (int w = 0; w < WARPS; ++w) {
          const float2 x = sh.part[w * S::ROWS + r];
          const float f = ex2(x.x - top);
          sum = fmaf(x.y, f, sum);
#pragma unroll
          for (int c = 0; c < N; ++c) y[c] = fmaf(sh.os[(w * S::ROWS + r) * VDIM + lane * N + c], f, y[c]);
        }
#pragma unroll
        for (int c = 0; c < N; ++c) a.ws[(slot * most + r) * VDIM + lane * N + c] = y[c];
        if (lane == 0) reinterpret_cast<float2*>(a.ws + slots * most * VDIM)[slot * most + r] = make_float2(top, sum);
      }
      __syncthreads();                                             // (before the next piece's rings and queries)
      u += to - from;
    }
  }
}

// Warp per (row, head): the parts that blocks c0 .. c1 have left of its history, always in the same order
template <int DIM, int VDIM> __global__ void __launch_bounds__(128) tree_attn4_join_kernel(const __grid_constant__ TreeArgs a) {
  constexpr int N = VDIM / 32;
  pdl_launch_dependents();
  pdl_wait();
  const int z = blockIdx.y, lane = threadIdx.x & 31, at = blockIdx.x * 4 + (threadIdx.x >> 5), i = at / a.H, h = at - i * a.H, most = a.rows * a.rep;
  const Portion p = portion_of(a, z);
  if (!p.held) {
    if (blockIdx.x == 0) nan_rows<VDIM>(a, p);
    return;
  }
  if (i >= p.n) return;
  const int g = h / a.rep, r = i * a.rep + h - g * a.rep;
  int lo;
  const int units = units_of(a, z, lo);
  long long before = 0, total = 0;                                 // units of the portions before, and of all
  for (int x = lane; x < a.nseg; x += 32) {
    int unused;
    const int n = units_of(a, x, unused);
    total += n;
    if (x < z) before += n;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    before += __shfl_xor_sync(0xffffffffu, before, o);
    total += __shfl_xor_sync(0xffffffffu, total, o);
  }
  const long long blocks = min((long long)a.spans, total);
  const int c0 = (int)(((before + 1) * blocks - 1) / total), c1 = (int)(((before + units) * blocks - 1) / total);            // (block c begins with unit total * c / blocks, rounded down)
  const long long slots = (long long)(a.nseg + a.spans) * a.G;
  auto slot = [&](int c) { return ((long long)(z + c) * a.G + g) * most + r; };
  const float2* ml = reinterpret_cast<const float2*>(a.ws + slots * most * VDIM);
  float top = -INFINITY;
  for (int c = c0 + lane; c <= c1; c += 32) top = fmaxf(top, ml[slot(c)].x);
  top = warp_max(top);
  const float base = top == -INFINITY ? 0.f : top;
  float o[N] = {}, l = 0.f;
#pragma unroll 4
  for (int c = c0; c <= c1; ++c) {
    const float2 x = ml[slot(c)];
    const float f = ex2(x.x - base);
    const float* src = a.ws + slot(c) * VDIM + lane * N;
    l = fmaf(x.y, f, l);
    float w[N];
    if constexpr (N == 4) *reinterpret_cast<float4*>(w) = *reinterpret_cast<const float4*>(src);
    else *reinterpret_cast<float2*>(w) = *reinterpret_cast<const float2*>(src);
#pragma unroll
    for (int e = 0; e < N; ++e) o[e] = fmaf(w[e], f, o[e]);
  }
  put_row<DIM, VDIM, LIA_CACHE_INT4>(a, p, i, h, o, l);
}

template <int DIM, int VDIM, int NR, bool PACKED> int launch(const TreeArgs& a, int nseg, cudaStream_t stream) {
  using S = Four<DIM, VDIM, NR>;
  static_assert(S::SMEM <= 232448 / tree_attn4_blocks(NR) - 1024, "shared memory");
  static bool configured[64] = {};                                 // per device
  int dev = 0;
  LIA_CUDA(cudaGetDevice(&dev));
  if (S::SMEM > 48 * 1024 && (dev >= 64 || !configured[dev])) {
    LIA_CUDA(cudaFuncSetAttribute(tree_attn4_kernel<DIM, VDIM, NR, PACKED>, cudaFuncAttributeMaxDynamicSharedMemorySize, S::SMEM));
    if (dev < 64) configured[dev] = true;
  }
  const dim3 grid(a.splits, a.tiles * a.G, nseg);
  if (a.splits > 1 && a.splits <= CLUSTER) LIA_CUDA(lia_launch_cluster(a.splits, tree_attn4_kernel<DIM, VDIM, NR, PACKED>, grid, dim3(THREADS), S::SMEM, stream, a));
  else LIA_CUDA(lia_launch(tree_attn4_kernel<DIM, VDIM, NR, PACKED>, grid, dim3(THREADS), S::SMEM, stream, a));
  return LIA_OK;
}
template <int DIM, int VDIM, bool PACKED> int launch_spans(const TreeArgs& a, int nseg, cudaStream_t stream) {
  static_assert(Four<DIM, VDIM, 1>::SMEM <= 48 * 1024, "shared memory");
  LIA_CUDA(lia_launch(tree_attn4_spans_kernel<DIM, VDIM, PACKED>, dim3(a.spans * a.G), dim3(THREADS), (size_t)Four<DIM, VDIM, 1>::SMEM, stream, a));
  LIA_CUDA(lia_launch(tree_attn4_join_kernel<DIM, VDIM>, dim3((unsigned)(((long long)a.rows * a.H + 3) / 4), nseg), dim3(128), 0, stream, a));
  return LIA_OK;
}
template <int DIM, int VDIM> int launch_rows(const TreeArgs& a, int nr, int nseg, cudaStream_t stream) {
  const bool packed = a.rows * a.rep <= 2;
  if (nr == 4) return launch<DIM, VDIM, 4, false>(a, nseg, stream);
  if (nr == 2) return launch<DIM, VDIM, 2, false>(a, nseg, stream);
  if (a.spans > 0) return packed ? launch_spans<DIM, VDIM, true>(a, nseg, stream) : launch_spans<DIM, VDIM, false>(a, nseg, stream);
  return packed ? launch<DIM, VDIM, 1, true>(a, nseg, stream) : launch<DIM, VDIM, 1, false>(a, nseg, stream);
}

}  // namespace

int lia_tree_attn_4bit(const void* args, int nr, int nseg, lia_stream_t stream_) {
  const TreeArgs& a = *reinterpret_cast<const TreeArgs*>(args);
  cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_);
  if (a.k.dim == 128) return a.v.dim == 128 ? launch_rows<128, 128>(a, nr, nseg, stream) : launch_rows<128, 64>(a, nr, nseg, stream);
  return a.v.dim == 128 ? launch_rows<64, 128>(a, nr, nseg, stream) : launch_rows<64, 64>(a, nr, nseg, stream);
}
