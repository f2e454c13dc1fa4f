// Rows of caches moved about: a request's history copied to other requests' slots (fork), and the tokens of a drafted tree that were accepted moved behind the history (compaction).  All tensors of
// all layers in one launch (in groups of MOST tensors), of any type and with positions anywhere among their dimensions, as bytes.
//
//   fork      slot `to` gets positions 0 .. count - 1 of slot `from`, and its whole state where a tensor has no positions.  A block brings 16 KB of a source once and writes it to every slot that is to
//             get it, two vectors a thread on their way at a time, four blocks an SM (with four vectors two blocks fit, 54 us instead of 48 for a prompt of 2049 tokens to 7 slots, 268 MB).
//   compact   position p0 + i of a portion's slot gets position p0 + kept[i], for ascending kept.  A thread has a column of the rows and takes them in order, eight at a time: kept[i] >= i, so what is
//             written (up to the i-th place) lies before all that is still to be read, and no two threads share a byte.
//
// Bound: fork by memory (every byte is read once and written once for each target), compaction by latency: a few rows in each of hundreds of tensors.
#include <algorithm>

#include "common.cuh"

namespace {

constexpr int MOST = 64, THREADS = 256, HELD = 2, CHUNK = 16384, BATCH = 8;
constexpr int COLUMNS = 64;                                        // threads of a block that compacts: a row is 32 to 128 vectors, scales 8 (with 256 threads 64 portions of 60 tensors took 9.9 us)

struct Tensor {
  uint8_t* data;
  long long slot, pos, piece;                                      // bytes from one to the next
  long long bytes;                                                 // of a piece (of a position)
  int pieces, vec;                                                 // vec: bytes that are moved at once
  int per, state;                                                  // positions of a chunk; state: how many positions a slot without any counts as
};
struct Tensors {
  Tensor t[MOST];
};

template <typename V>
__device__ __forceinline__ void fork_chunk_of(const Tensor& t, const int* copies, int c, int n, int slots, int most, int capacity, long long first) {
  const int end = (int)min((long long)t.per, (long long)most - first);                         // positions of this chunk
  const unsigned vpp = (unsigned)(t.bytes / sizeof(V)), run = t.pos == t.bytes ? (unsigned)end * vpp : vpp, outer = t.pos == t.bytes ? (unsigned)t.pieces : (unsigned)(end * t.pieces);
  const uint8_t* src = t.data + copies[3 * c] * t.slot + first * t.pos;
  for (unsigned v0 = threadIdx.x; v0 < run * outer; v0 += THREADS * HELD) {
    V held[HELD];
    long long at[HELD];
    int pos[HELD];
#pragma unroll
    for (int i = 0; i < HELD; ++i) {
      const unsigned v = v0 + i * THREADS;
      pos[i] = -1;
      if (v >= run * outer) continue;
      const unsigned o = v / run, x = v - o * run;
      if (t.pos == t.bytes) {                                      // positions side by side inside each piece
        at[i] = o * t.piece + (long long)x * sizeof(V);
        pos[i] = (int)(x / vpp);
      } else {
        const unsigned p = o / (unsigned)t.pieces;
        at[i] = p * t.pos + (o - p * t.pieces) * t.piece + (long long)x * sizeof(V);
        pos[i] = (int)p;
      }
      held[i] = __ldcg(reinterpret_cast<const V*>(src + at[i]));
    }
    for (int j = c; j < n; ++j) {
      const int from = copies[3 * j], to = copies[3 * j + 1], count = t.state > 0 ? t.state : min(copies[3 * j + 2], capacity);
      if (from != copies[3 * c] || (unsigned)to >= (unsigned)slots || to == from) continue;
      uint8_t* dst = t.data + to * t.slot + first * t.pos;
#pragma unroll
      for (int i = 0; i < HELD; ++i)
        if (pos[i] >= 0 && first + pos[i] < count) *reinterpret_cast<V*>(dst + at[i]) = held[i];
    }
  }
}

// (apart, so that the narrow ones do not cost the wide one registers)
template <typename V> __device__ __noinline__ void fork_chunk(const Tensor& t, const int* copies, int c, int n, int slots, int most, int capacity, long long first) {
  fork_chunk_of<V>(t, copies, c, n, slots, most, capacity, first);
}

// Grid: copies, chunks of positions, tensors
__global__ void __launch_bounds__(THREADS, 4) cache_fork_kernel(const __grid_constant__ Tensors all, const int* __restrict__ copies, int n, int slots, int capacity) {
  pdl_launch_dependents();
  pdl_wait();
  const Tensor& t = all.t[blockIdx.z];
  const int c = blockIdx.x, from = copies[3 * c];
  if ((unsigned)from >= (unsigned)slots) return;
  for (int j = 0; j < c; ++j)
    if (copies[3 * j] == from) return;                             // that copy's block takes all targets of the source
  int most = t.state;
  if (t.state == 0)
    for (int j = c; j < n; ++j)
      if (copies[3 * j] == from) most = max(most, min(copies[3 * j + 2], capacity));
  for (long long first = (long long)blockIdx.y * t.per; first < most; first += (long long)gridDim.y * t.per) {
    switch (t.vec) {
      case 16: fork_chunk_of<uint4>(t, copies, c, n, slots, most, capacity, first); break;
      case 8: fork_chunk<uint2>(t, copies, c, n, slots, most, capacity, first); break;
      case 4: fork_chunk<uint32_t>(t, copies, c, n, slots, most, capacity, first); break;
      case 2: fork_chunk<uint16_t>(t, copies, c, n, slots, most, capacity, first); break;
      default: fork_chunk<uint8_t>(t, copies, c, n, slots, most, capacity, first);
    }
  }
}

template <typename V>
__device__ __forceinline__ void compact_column(const Tensor& t, uint8_t* base, const int* kept, int most, int n, unsigned column) {
  const unsigned vpp = (unsigned)(t.bytes / sizeof(V)), piece = column / vpp;
  uint8_t* at = base + piece * t.piece + (long long)(column - piece * vpp) * sizeof(V);
  int last = -1;
  for (int i0 = 0; i0 < most; i0 += BATCH) {
    V held[BATCH];
    int from[BATCH];
#pragma unroll
    for (int i = 0; i < BATCH; ++i) {
      from[i] = -1;
      if (i0 + i >= most || last == n) continue;
      const int k = kept[i0 + i];
      if (k <= last || k >= n) {                                   // the list's end
        last = n;
        continue;
      }
      last = k;
      from[i] = k;
      if (k != i0 + i) held[i] = __ldcg(reinterpret_cast<const V*>(at + k * t.pos));
    }
#pragma unroll
    for (int i = 0; i < BATCH; ++i)
      if (from[i] >= 0 && from[i] != i0 + i) *reinterpret_cast<V*>(at + (i0 + i) * t.pos) = held[i];
    if (last == n) return;
  }
}

// Grid: columns of the rows, tensors, portions
__global__ void __launch_bounds__(COLUMNS) cache_compact_kernel(const __grid_constant__ Tensors all, const int* __restrict__ segs, const int* __restrict__ kept, int most, int slots, int capacity) {
  pdl_launch_dependents();
  pdl_wait();
  const Tensor& t = all.t[blockIdx.y];
  const int* s = segs + 4ll * blockIdx.z;
  const int slot = s[0], p0 = s[1], n = s[3];
  if ((unsigned)slot >= (unsigned)slots || p0 < 0 || n <= 0 || n > capacity || p0 > capacity - n) return;
  const unsigned column = blockIdx.x * COLUMNS + threadIdx.x;
  if (column >= (unsigned)(t.bytes / t.vec) * (unsigned)t.pieces) return;
  uint8_t* base = t.data + slot * t.slot + p0 * t.pos;
  const int* list = kept + (long long)blockIdx.z * most;
  switch (t.vec) {
    case 16: compact_column<uint4>(t, base, list, most, n, column); break;
    case 8: compact_column<uint2>(t, base, list, most, n, column); break;
    case 4: compact_column<uint32_t>(t, base, list, most, n, column); break;
    case 2: compact_column<uint16_t>(t, base, list, most, n, column); break;
    default: compact_column<uint8_t>(t, base, list, most, n, column);
  }
}

// NULL, or what is wrong with a tensor; else how the kernels take it
const char* tensor_of(const LiaCacheRows& r, int slots, int capacity, Tensor& t) {
  if (!r.data) return "null tensor";
  if (r.pieces <= 0 || r.piece_bytes <= 0 || (long long)r.pieces * r.piece_bytes >= 1ll << 31) return "rows of no or too many bytes";
  if (r.state && r.pieces != 1) return "a state in pieces";
  // each of slots, positions and pieces steps over all that lies closer together
  struct Step {
    long long stride, n;
  } steps[3] = {{r.slot_stride, slots}, {r.pos_stride, r.state ? 1 : capacity}, {r.piece_stride, r.pieces}};
  std::sort(steps, steps + 3, [](const Step& a, const Step& b) { return a.stride < b.stride; });
  __int128 span = r.piece_bytes;
  for (const Step& s : steps) {
    if (s.n <= 1) continue;
    if (s.stride < span) return "slots or rows that share their place";
    span += (__int128)(s.n - 1) * s.stride;
  }
  t = Tensor{static_cast<uint8_t*>(r.data), r.slot_stride, r.pos_stride, r.piece_stride, r.piece_bytes, r.pieces, 16, 1, 0};
  const uintptr_t bits = reinterpret_cast<uintptr_t>(r.data) | (uintptr_t)r.slot_stride | (r.state ? 0 : (uintptr_t)r.pos_stride) | (r.pieces > 1 ? (uintptr_t)r.piece_stride : 0) | (uintptr_t)r.piece_bytes;
  while (bits % t.vec) t.vec /= 2;
  if (r.state) {                                                   // a slot's bytes as positions of one vector each
    t.state = (int)(r.piece_bytes / t.vec);
    t.pos = t.bytes = t.vec;
  }
  const long long row = t.bytes * t.pieces;
  t.per = (int)(row >= CHUNK ? 1 : CHUNK / row);
  return nullptr;
}

}  // namespace

extern "C" int lia_cache_fork(const LiaCacheRows* tensors, int n_tensors, int slots, int capacity, const int* copies, int n, int max_count, lia_stream_t stream) {
  LIA_CHECK_ARG(n_tensors >= 0 && slots > 0 && capacity > 0 && n >= 0, "lia_cache_fork: bad sizes");
  if (n_tensors == 0 || n == 0) return LIA_OK;
  LIA_CHECK_ARG(tensors && copies, "lia_cache_fork: null pointer");
  for (int t0 = 0; t0 < n_tensors; t0 += MOST) {
    Tensors all;
    const int m = n_tensors - t0 < MOST ? n_tensors - t0 : MOST;
    long long chunks = 1;
    for (int i = 0; i < m; ++i) {
      const char* wrong = tensor_of(tensors[t0 + i], slots, capacity, all.t[i]);
      LIA_CHECK_ARG(!wrong, "lia_cache_fork: %s", wrong);
      const long long positions = all.t[i].state > 0 ? all.t[i].state : max_count < 1 ? 1 : max_count < capacity ? max_count : capacity, need = (positions + all.t[i].per - 1) / all.t[i].per;
      if (need > chunks) chunks = need;
    }
    LIA_CUDA(lia_launch(cache_fork_kernel, dim3(n, (unsigned)(chunks < 16384 ? chunks : 16384), m), dim3(THREADS), 0, reinterpret_cast<cudaStream_t>(stream), all, copies, n, slots, capacity));
  }
  return LIA_OK;
}

extern "C" int lia_cache_compact(const LiaCacheRows* tensors, int n_tensors, int slots, int capacity, const int* segs, int nseg, const int* kept, int most, lia_stream_t stream) {
  LIA_CHECK_ARG(n_tensors >= 0 && slots > 0 && capacity > 0 && nseg >= 0 && most >= 0, "lia_cache_compact: bad sizes");
  if (n_tensors == 0 || nseg == 0 || most == 0) return LIA_OK;
  LIA_CHECK_ARG(tensors && segs && kept, "lia_cache_compact: null pointer");
  LIA_CHECK_ARG(nseg <= 65535, "lia_cache_compact: too many portions");
  for (int t0 = 0; t0 < n_tensors; t0 += MOST) {
    Tensors all;
    const int m = n_tensors - t0 < MOST ? n_tensors - t0 : MOST;
    long long columns = 1;
    for (int i = 0; i < m; ++i) {
      const char* wrong = tensor_of(tensors[t0 + i], slots, capacity, all.t[i]);
      LIA_CHECK_ARG(!wrong, "lia_cache_compact: %s", wrong);
      LIA_CHECK_ARG(!tensors[t0 + i].state, "lia_cache_compact: a state has no positions");
      const long long c = all.t[i].bytes / all.t[i].vec * all.t[i].pieces;
      if (c > columns) columns = c;
    }
    LIA_CUDA(lia_launch(cache_compact_kernel, dim3((unsigned)((columns + COLUMNS - 1) / COLUMNS), m, nseg), dim3(COLUMNS), 0, reinterpret_cast<cudaStream_t>(stream), all, segs, kept, most, slots,
                        capacity));
  }
  return LIA_OK;
}
