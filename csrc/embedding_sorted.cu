// Embedding lookup with scaling, and its gradient by sorted tokens.
//
//   out[i] = scale * W[idx_i]        dW[v] = scale * sum over {i : idx_i = v} of dout[i]
//
// The sum of a row is taken in fp32 in an order that depends on the tokens of the
// call alone: the positions are sorted by token (stable, so ascending within a
// token), the sorted list of all tokens is cut into chunks of 32 entries, and every
// run of one token is summed front to back inside a chunk; a run that crosses
// chunks leaves one fp32 partial per chunk, added up in chunk order (by eighths of
// the chunks where there are many).  No atomics touch values, so the gradient is
// the same from run to run, and no [V, C] accumulator is kept.
//
// The lookup sorts for the backward pass on one cluster while the other SMs
// gather.  Tokens outside [0, V) read as a zero row; they and the padding token
// get no gradient (key V, sorted behind all others).
#include <cooperative_groups.h>

#include <algorithm>
#include <utility>

#include "common.cuh"
#include "vec.cuh"

namespace msb {

MSB_BOUNDS_TU(embedding)

namespace {

namespace cg = cooperative_groups;

// Entries that a warp sums.  With 8, 16384 x 768 naturally distributed tokens took
// 25 us instead of 27, but 65536 of them 68 instead of 47 and 65536 times one token
// 385 instead of 86: the shorter the chunks, the more parts of cut runs.
constexpr int kChunk = 32;
constexpr int kSortThreads = 1024;
constexpr int kDigit = 9;           // most bits of a sorting pass
constexpr int kBins = 1 << kDigit;
constexpr int kSortWarps = kSortThreads / 32;
constexpr int kMaxCluster = 8;   // 16 blocks sort 16384 tokens in 12 us, but are not portable
constexpr int kHeld = 4;            // entries a lane keeps in registers over a pass
constexpr int kRows = 4;            // rows in flight in the sum kernel (8: 65536 x 768 54 us, 4: 47)

// Eight columns of a row as a lane holds them: packed while in flight.  VEC:
// adjacent columns from c0 on; otherwise c0 + 32 k, for widths and addresses that
// do not allow 16-byte accesses.
template <typename T, bool VEC>
struct Cols {
  uint4 r[sizeof(T) == 4 ? 2 : 1];
  T e[VEC ? 1 : 8];
  __device__ __forceinline__ void load(const T* row, int c0, int C) {
    if constexpr (VEC) {
#pragma unroll
      for (int k = 0; k < (int)(sizeof(T) == 4 ? 2 : 1); ++k)
        r[k] = c0 < C ? reinterpret_cast<const uint4*>(row + c0)[k] : make_uint4(0, 0, 0, 0);
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k) e[k] = c0 + 32 * k < C ? row[c0 + 32 * k] : from_f32<T>(0.f);
    }
  }
  __device__ __forceinline__ void numbers(float (&f)[8]) const {
    if constexpr (!VEC) {
#pragma unroll
      for (int k = 0; k < 8; ++k) f[k] = to_f32(e[k]);
    } else if constexpr (sizeof(T) == 2) {
      unpack_u4<T>(r[0], f);
    } else {
      const uint4 a = r[0], b = r[sizeof(T) == 4 ? 1 : 0];
      f[0] = __uint_as_float(a.x), f[1] = __uint_as_float(a.y), f[2] = __uint_as_float(a.z),
      f[3] = __uint_as_float(a.w), f[4] = __uint_as_float(b.x), f[5] = __uint_as_float(b.y),
      f[6] = __uint_as_float(b.z), f[7] = __uint_as_float(b.w);
    }
  }
  static __device__ __forceinline__ void store(T* row, int c0, int C, const float (&f)[8]) {
    if constexpr (!VEC) {
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (c0 + 32 * k < C) row[c0 + 32 * k] = from_f32<T>(f[k]);
    } else {
      if (c0 >= C) return;
      if constexpr (sizeof(T) == 2) {
        *reinterpret_cast<uint4*>(row + c0) = pack_u4<T>(f);
      } else {
        reinterpret_cast<float4*>(row + c0)[0] = make_float4(f[0], f[1], f[2], f[3]);
        reinterpret_cast<float4*>(row + c0)[1] = make_float4(f[4], f[5], f[6], f[7]);
      }
    }
  }
};

// out = scale * w[idx], from thread `first` of `threads` on.  VEC: eight columns a
// thread (width a multiple of 8, 16-byte aligned table).
template <typename T, bool VEC>
__device__ __forceinline__ void lookup(const long long* __restrict__ idx,
                                       const T* __restrict__ w, T* __restrict__ out,
                                       unsigned total, const FastDiv& per, int C, long long V,
                                       float scale, unsigned first, unsigned threads) {
  constexpr int U = 4;   // in flight
  for (unsigned i0 = first; i0 < total; i0 += U * threads) {
    Cols<T, true> v[U];
    T e[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const unsigned i = i0 + u * threads;
      const bool live = i < total;   // a place behind the end has column 0 of no token
      const unsigned m = live ? per.div(i) : 0u;
      const int c = live ? (int)(i - m * per.d) * (VEC ? 8 : 1) : 0;
      const long long t = live ? idx[m] : -1;
      const bool in = t >= 0 && t < V;
      if (c == 0 && live) (void)MSB_OK(in, kSiteEmbeddingToken, t, V);
      if constexpr (VEC) {
        v[u].load(w + (in ? t : 0) * C, c, in ? C : 0);   // zeros where not in
      } else {
        e[u] = in ? w[t * C + c] : from_f32<T>(0.f);
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const unsigned i = i0 + u * threads;
      if (i >= total) continue;
      if constexpr (VEC) {   // rows lie one behind the other
        float f[8];
        v[u].numbers(f);
#pragma unroll
        for (int k = 0; k < 8; ++k) f[k] *= scale;
        Cols<T, true>::store(out + (long long)i * 8, 0, 8, f);
      } else {
        out[i] = from_f32<T>(to_f32(e[u]) * scale);
      }
    }
  }
}

template <typename T, bool VEC>
__global__ void __launch_bounds__(256)
lookup_kernel(const long long* __restrict__ idx, const T* __restrict__ w, T* __restrict__ out,
              unsigned total, FastDiv per, int C, long long V, float scale) {
  ::msb::pdl_begin();
  lookup<T, VEC>(idx, w, out, total, per, C, V, scale, blockIdx.x * blockDim.x + threadIdx.x,
                 gridDim.x * blockDim.x);
}

// Sorts (token, position) by token on one cluster, 9 bits or fewer a pass.
//
// Every warp of the cluster owns one contiguous piece of the list.  A pass
// counts the digits of each warp's piece, turns the counts into places (over
// the warps of a block, over the blocks, each of which writes its totals into
// the others' shared memory, over the digits), and writes each entry to its
// place, warp by warp in order, lanes with the same digit ranked by ballots on
// its bits (__match_any_sync took seven times as long): stable by construction.
// The cluster barrier orders the passes.  What bounds it is the latency of its
// steps: 16384 tokens of 50257 take 13 us.
__device__ __forceinline__ void sort_tokens(const long long* __restrict__ idx, long long n,
                                            long long V, long long padding, int passes, int bits,
                                            uint2* list_a, uint2* list_b) {
  extern __shared__ unsigned cnt[];   // [kSortWarps][1 << bits]
  __shared__ unsigned hist[kMaxCluster][kBins], base[kBins], wsum[kSortWarps], quarter[4][kBins];
  cg::cluster_group cluster = cg::this_cluster();
  const unsigned q = cluster.block_rank(), R = cluster.num_blocks();
  auto started = cluster.barrier_arrive();   // waited for before another block's memory is written
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int bins = 1 << bits;
  const unsigned ones = (unsigned)bins - 1u, below = (1u << lane) - 1u;
  const long long per = (n + (long long)R * kSortThreads - 1) / ((long long)R * kSortThreads) * 32;
  const long long lo = min(n, per * (q * kSortWarps + warp)), hi = min(n, lo + per);
  unsigned* mine = cnt + warp * bins;
  auto load = [&](int p, long long i) {   // (token, position) of entry i
    if (i >= hi) return make_uint2(0u, 0u);
    if (p > 0) return __ldcg((p & 1 ? list_a : list_b) + i);   // other blocks wrote it
    const long long t = idx[i];
    return make_uint2(t >= 0 && t < V && t != padding ? (unsigned)t : (unsigned)V, (unsigned)i);
  };
  for (int p = 0; p < passes; ++p) {
    const int shift = p * bits;
    uint2 held[kHeld];
    unsigned same[kHeld];
#pragma unroll
    for (int h = 0; h < kHeld; ++h) held[h] = load(p, lo + h * 32 + lane);
    for (int b = lane * 4; b < bins; b += 128)
      *reinterpret_cast<uint4*>(mine + b) = make_uint4(0, 0, 0, 0);
    __syncwarp();
    auto match = [&](unsigned key, long long i) {   // the lanes with this lane's digit
      const unsigned d = (key >> shift) & ones;
      unsigned m = __ballot_sync(0xffffffffu, i < hi);
#pragma unroll
      for (int b = 0; b < kDigit; ++b) {   // bits from `bits` on are 0 everywhere
        const bool set = d >> b & 1;
        const unsigned v = __ballot_sync(0xffffffffu, set);
        m &= set ? v : ~v;
      }
      return m;
    };
    auto count = [&](unsigned key, long long i, unsigned m) {
      if (i < hi && (m & below) == 0) mine[(key >> shift) & ones] += __popc(m);
      __syncwarp();
    };
#pragma unroll
    for (int h = 0; h < kHeld; ++h) {
      if (lo + h * 32 < hi) {
        same[h] = match(held[h].x, lo + h * 32 + lane);
        count(held[h].x, lo + h * 32 + lane, same[h]);
      }
    }
    for (long long i0 = lo + kHeld * 32; i0 < hi; i0 += 32) {
      const unsigned key = load(p, i0 + lane).x;
      count(key, i0 + lane, match(key, i0 + lane));
    }
    __syncthreads();
    // where each warp's entries of a digit begin among the block's: sums over
    // the warps, a quarter of them a thread
    for (int t = threadIdx.x; t < 4 * bins; t += kSortThreads) {
      const int d = t & (bins - 1), part = t >> bits;
      unsigned run = 0;
#pragma unroll
      for (int w = 0; w < kSortWarps / 4; ++w) {
        unsigned* at = cnt + (part * (kSortWarps / 4) + w) * bins + d;
        const unsigned v = *at;
        *at = run;
        run += v;
      }
      quarter[part][d] = run;
    }
    __syncthreads();
    if (p == 0) cluster.barrier_wait(std::move(started));
    if (threadIdx.x < bins) {
      unsigned run = 0;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const unsigned v = quarter[k][threadIdx.x];
        quarter[k][threadIdx.x] = run;
        run += v;
      }
      for (unsigned r = 0; r < R; ++r)
        cluster.map_shared_rank(&hist[0][0], r)[q * kBins + threadIdx.x] = run;
    }
    cluster.sync();
    unsigned before = 0, all = 0;
    if (threadIdx.x < bins) {
#pragma unroll
      for (unsigned r = 0; r < kMaxCluster; ++r) {
        const unsigned v = r < R ? hist[r][threadIdx.x] : 0u;
        before += r < q ? v : 0u;
        all += v;
      }
    }
    unsigned incl = all;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const unsigned v = __shfl_up_sync(0xffffffffu, incl, o);
      incl += lane >= o ? v : 0u;
    }
    if (lane == 31) wsum[warp] = incl;
    __syncthreads();
    const unsigned lower = __reduce_add_sync(0xffffffffu, lane < warp ? wsum[lane] : 0u);
    if (threadIdx.x < bins) base[threadIdx.x] = lower + incl - all + before;
    __syncthreads();
    uint2* out = p & 1 ? list_b : list_a;
    const unsigned* ahead = quarter[warp / (kSortWarps / 4)];
    auto place = [&](uint2 e, long long i, unsigned m) {
      const unsigned d = (e.x >> shift) & ones;
      if (i < hi) out[base[d] + ahead[d] + mine[d] + __popc(m & below)] = e;
      __syncwarp();
      if (i < hi && (m & below) == 0) mine[d] += __popc(m);
      __syncwarp();
    };
#pragma unroll
    for (int h = 0; h < kHeld; ++h) {
      if (lo + h * 32 < hi) place(held[h], lo + h * 32 + lane, same[h]);
    }
    for (long long i0 = lo + kHeld * 32; i0 < hi; i0 += 32) {
      const uint2 e = load(p, i0 + lane);
      place(e, i0 + lane, match(e.x, i0 + lane));
    }
    cluster.sync();   // the list is written, and hist may be again
  }
}

// The first cluster sorts, the others gather.
template <typename T, bool VEC>
__global__ void __launch_bounds__(kSortThreads)
lookup_sort_kernel(const long long* __restrict__ idx, const T* __restrict__ w,
                   T* __restrict__ out, unsigned total, FastDiv per, int C, long long V,
                   float scale, long long n, long long padding, int passes, int bits,
                   uint2* list_a, uint2* list_b) {
  ::msb::pdl_begin();
  const unsigned R = cg::this_cluster().num_blocks();
  if (blockIdx.x < R) {
    sort_tokens(idx, n, V, padding, passes, bits, list_a, list_b);
  } else {
    lookup<T, VEC>(idx, w, out, total, per, C, V, scale,
                   (blockIdx.x - R) * kSortThreads + threadIdx.x,
                   (gridDim.x - R) * kSortThreads);
  }
}

// Clears the rows of a unit of `unit` table rows that no entry of the list names.
constexpr int kUnitRows = 1024;
template <typename T, bool VEC>
__device__ __forceinline__ void clear_unit(const uint2* __restrict__ list, long long n,
                                           long long V, int C, T* grad, long long u, int unit) {
  __shared__ unsigned char named[kUnitRows];
  const long long v0 = u * unit, v1 = min(V, v0 + unit);
  for (int i = threadIdx.x; i < unit; i += blockDim.x) named[i] = 0;
  // the first entry that is not before v0: all threads probe, 256 places at a time
  long long lo = 0, hi = n;
  while (lo < hi) {
    const long long step = (hi - lo + blockDim.x - 1) / blockDim.x;
    const long long at = lo + threadIdx.x * step;
    const int before = __syncthreads_count(at < hi && list[at].x < v0);
    if (before == 0) break;             // list[lo] is not before v0
    hi = min(hi, lo + before * step);   // nor is list[lo + before * step]
    lo += (before - 1) * step + 1;
  }
  for (;;) {   // mark the unit's
    const long long at = lo + threadIdx.x;
    const unsigned k = at < n ? list[at].x : 0xffffffffu;
    if (k < v1) named[k - v0] = 1;
    if (__syncthreads_count(k < v1) < (int)blockDim.x) break;
    lo += blockDim.x;
  }
  T* g = grad + v0 * C;
  if (VEC) {
    constexpr int N = 16 / sizeof(T);
    const int per = C / N, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    for (int r = warp; r < v1 - v0; r += blockDim.x >> 5) {
      if (named[r]) continue;
      uint4* p = reinterpret_cast<uint4*>(g + (long long)r * C);
      for (int i = lane; i < per; i += 32) p[i] = make_uint4(0, 0, 0, 0);
    }
  } else {
    for (int r = 0; r < v1 - v0; ++r) {
      if (named[r]) continue;
      for (int c = threadIdx.x; c < C; c += blockDim.x) g[(long long)r * C + c] = from_f32<T>(0.f);
    }
  }
}

// A warp sums a chunk of the list over 256 columns.  The rows of four entries, and
// the gradient rows that their sums are added to, are loaded before any is used,
// whatever runs they belong to: most runs are one or two entries long, and run by
// run the loads would wait for one another.  open[j]: a run begins in chunk j and
// goes on behind it.
//
// ADD: the sums are added to the rows.  Otherwise the gradient is a new one, and
// the blocks behind the first `row_blocks` clear the rows of no token meanwhile.
template <typename T, bool VEC, bool ADD>
__global__ void __launch_bounds__(256)
sorted_rows_kernel(const uint2* __restrict__ list, long long n, unsigned V,
                   const T* __restrict__ dout, int C, FastDiv slabs, unsigned tasks, T* grad,
                   float scale, float* __restrict__ part, unsigned char* __restrict__ open,
                   unsigned row_blocks, int unit) {
  ::msb::pdl_begin();
  if (!ADD && blockIdx.x >= row_blocks) {
    clear_unit<T, VEC>(list, n, V, C, grad, blockIdx.x - row_blocks, unit);
    return;
  }
  const int lane = threadIdx.x & 31;
  const unsigned task = blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
  if (task >= tasks) return;
  const unsigned j = slabs.div(task);
  const long long first = (long long)j * kChunk;
  const int c0 = (int)(task - j * slabs.d) * 256 + (VEC ? lane * 8 : lane);
  const int len = (int)min((long long)kChunk, n - first);
  // lane l: entry l's token; what comes before and behind the chunk
  const uint2 entry = lane < len ? list[first + lane] : make_uint2(V, 0u);
  const unsigned my_key = entry.x, my_pos = entry.y;
  const unsigned prev = first > 0 ? list[first - 1].x : V;
  const unsigned next = first + kChunk < n ? list[first + kChunk].x : V;
  unsigned behind = __shfl_down_sync(0xffffffffu, my_key, 1);   // the key after each entry
  if (lane == kChunk - 1) behind = next;
  // entries that are tokens, and those that end a run inside the chunk
  const unsigned live = __ballot_sync(0xffffffffu, lane < len && my_key < V);
  const unsigned ends = __ballot_sync(0xffffffffu, lane < len && my_key < V && behind != my_key);
  if (c0 == 0) open[j] = live >> (kChunk - 1) & 1 && !(ends >> (kChunk - 1) & 1);   // goes on
  if (live == 0) return;
  const unsigned key0 = __shfl_sync(0xffffffffu, my_key, 0);
  const int head = prev == key0 ? __ffs(~__ballot_sync(0xffffffffu, my_key == key0)) - 1 : 0;
  // `head` entries, when not 0, continue the run of the chunk before (32 of 32: -1)
  const unsigned in_head = prev != key0 ? 0u : head < 0 ? ~0u : (1u << head) - 1u;
  if (c0 == 0 && (in_head >> (kChunk - 1) & 1)) open[j] = 0;   // but began earlier
  float a[8] = {0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll 1
  for (int e0 = 0; e0 < kChunk; e0 += kRows) {
    if ((live >> e0) == 0) break;
    Cols<T, VEC> row[kRows], old[ADD ? kRows : 1];
#pragma unroll
    for (int u = 0; u < kRows; ++u) {
      const int e = e0 + u;
      const unsigned p = __shfl_sync(0xffffffffu, my_pos, e);
      const unsigned k = __shfl_sync(0xffffffffu, my_key, e);
      if (live >> e & 1) row[u].load(dout + (long long)p * C, c0, C);
      if (ADD && (ends >> e & 1) && !(in_head >> e & 1)) old[u].load(grad + (long long)k * C, c0, C);
    }
#pragma unroll
    for (int u = 0; u < kRows; ++u) {
      const int e = e0 + u;
      if (!(live >> e & 1)) break;
      float f[8];
      row[u].numbers(f);
#pragma unroll
      for (int k = 0; k < 8; ++k) a[k] += f[k];
      const bool end = ends >> e & 1, last = e == len - 1;
      if (!end && !last) continue;
      if (end && !(in_head >> e & 1)) {   // a whole run
        const unsigned k = __shfl_sync(0xffffffffu, my_key, e);
        if (ADD) {
          old[u].numbers(f);
#pragma unroll
          for (int i = 0; i < 8; ++i) f[i] = fmaf(a[i], scale, f[i]);
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i) f[i] = a[i] * scale;
        }
        Cols<T, VEC>::store(grad + (long long)k * C, c0, C, f);
      } else {   // a part: slot 0 continues the chunk before, slot 1 begins here
        Cols<float, VEC>::store(part + ((long long)j * 2 + (in_head >> e & 1 ? 0 : 1)) * C, c0, C,
                                a);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) a[i] = 0.f;
    }
  }
}

// Adds up the runs that go on behind the chunk they begin in.  A block has 32
// chunks and 128 columns; each of its warps takes every eighth open run among
// them and adds its parts in order, and runs of more than kLongRun parts, left
// for last, are added by the eight warps together, an eighth of the parts each,
// the eight sums in order.  V4: C is a multiple of 4.
constexpr int kRunThreads = 256;
constexpr int kRunWarps = kRunThreads / 32;
constexpr int kRunCols = 128;
constexpr int kLongRun = 24;
static_assert(kLongRun < 32, "a warp's one look finds the end of a short run");
template <typename T, bool ADD, bool V4>
__global__ void __launch_bounds__(kRunThreads)
sorted_runs_kernel(const uint2* __restrict__ list, long long n, const float* __restrict__ part,
                   int C, long long chunks, FastDiv slabs, T* grad, float scale,
                   const unsigned char* __restrict__ open) {
  ::msb::pdl_begin();
  __shared__ float4 sums[kRunWarps][32];
  __shared__ unsigned is_long;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const unsigned group = slabs.div(blockIdx.x);
  const int c = (int)(blockIdx.x - group * slabs.d) * kRunCols + lane * 4;
  const long long j0 = (long long)group * 32;
  unsigned todo = __ballot_sync(0xffffffffu, j0 + lane < chunks && open[j0 + lane]);
  if (todo == 0) return;   // in all warps alike
  if (threadIdx.x == 0) is_long = 0;
  __syncthreads();
  auto load = [&](const float* row) {
    if (V4) return c < C ? *reinterpret_cast<const float4*>(row + c) : make_float4(0, 0, 0, 0);
    return make_float4(c < C ? row[c] : 0.f, c + 1 < C ? row[c + 1] : 0.f,
                       c + 2 < C ? row[c + 2] : 0.f, c + 3 < C ? row[c + 3] : 0.f);
  };
  auto add_parts = [&](float4& a, long long j, int i0, int i1) {   // of chunks j + 1 + i
    const float* p = part + (j + 1) * 2 * C;
#pragma unroll 8
    for (int i = i0; i < i1; ++i) {
      const float4 v = load(p + (long long)i * 2 * C);
      a.x += v.x, a.y += v.y, a.z += v.z, a.w += v.w;
    }
  };
  auto put = [&](const float4& a, unsigned key) {
    T* g = grad + (long long)key * C + c;
    const float f[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (c + k < C) g[k] = from_f32<T>(fmaf(f[k], scale, ADD ? to_f32(g[k]) : 0.f));
  };
  for (int t = 0; todo != 0; ++t, todo &= todo - 1) {
    if (t % kRunWarps != warp) continue;
    const int b = __ffs(todo) - 1;
    const long long j = j0 + b, at = (j + 1 + lane) * kChunk;   // the chunks behind j
    const unsigned key = list[j * kChunk + kChunk - 1].x;
    const unsigned other = ~__ballot_sync(0xffffffffu, at < n && list[at].x == key);
    const int count = other == 0 ? 32 : __ffs(other) - 1;
    if (count > kLongRun) {
      if (lane == 0) atomicOr(&is_long, 1u << b);
      continue;
    }
    float4 a = load(part + (j * 2 + 1) * C);
    add_parts(a, j, 0, count);
    put(a, key);
  }
  __syncthreads();
  for (unsigned rest = is_long; rest != 0; rest &= rest - 1) {
    const long long j = j0 + __ffs(rest) - 1;
    const unsigned key = list[j * kChunk + kChunk - 1].x;
    long long count = 0;
    for (;;) {
      const long long at = (j + 1 + count + threadIdx.x) * kChunk;
      const int more = __syncthreads_count(at < n && list[at].x == key);
      count += more;
      if (more < kRunThreads) break;
    }
    const int each = (int)((count + kRunWarps - 1) / kRunWarps);
    const int i0 = min((int)count, each * warp), i1 = min((int)count, i0 + each);
    float4 a = warp == 0 ? load(part + (j * 2 + 1) * C) : make_float4(0.f, 0.f, 0.f, 0.f);
    add_parts(a, j, i0, i1);
    sums[warp][lane] = a;
    __syncthreads();
    if (warp == 0) {
#pragma unroll
      for (int w = 1; w < kRunWarps; ++w) {
        const float4 v = sums[w][lane];
        a.x += v.x, a.y += v.y, a.z += v.z, a.w += v.w;
      }
      put(a, key);
    }
    __syncthreads();   // sums may be written again
  }
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

long long chunks_of(long long n) { return (n + kChunk - 1) / kChunk; }

// Whether the lookup is launched by itself before the sort.  Beside the sort, a
// block a SM gathers at 2.6 TB/s of output, by itself the lookup does at 4.2;
// the sort takes some 9 us and 0.5 us for every 1000 tokens.  65536 x 4096 bf16:
// 207 us together, 163 apart; 65536 x 768: 43 us together, some 65 apart.
bool apart(long long n, long long bytes) { return bytes / 7e6 > 9 + n / 1900.0; }

}  // namespace

// the list that the backward needs is in the first 2 n words of `ws`, which has
// 4 n (null: not wanted)
void scaled_embedding_fwd(const long long* idx, const void* w, void* out, long long n, int C,
                          long long V, float scale, long long padding, unsigned* ws, int dtype,
                          cudaStream_t st) {
  if (n == 0) return;
  MSB_DISPATCH_FLOAT(dtype, T, {
    const bool vec = C % 8 == 0 && aligned16(w);
    const int per = vec ? C / 8 : C;
    const long long fit = (1LL << 30) / per, most = fit > 0 ? fit : 1;   // tokens a launch
    for (long long i = 0; i < n; i += most) {
      const unsigned total = (unsigned)((n - i < most ? n - i : most) * per);
      if (ws != nullptr && i == 0) {
        // tokens and V itself (no token) in as few passes of at most kDigit bits;
        // at least 2: a warp's counters are then whole vectors
        int total_bits = 2;
        while ((V >> total_bits) != 0) ++total_bits;
        const int passes = (total_bits + kDigit - 1) / kDigit;
        const int bits = max(2, (total_bits + passes - 1) / passes);
        unsigned R = 1;
        while (R < kMaxCluster && (long long)R * kSortThreads < n) R *= 2;
        // a block a SM in all: 64 registers a thread allow no more
        const bool alone = n > most || apart(n, n * C * (long long)sizeof(T));
        const unsigned gather =
            alone ? 0 : max(R, grid_for(total, kSortThreads, kNumSMs - R) / R * R);
        uint2 *a = (uint2*)ws, *b = (uint2*)(ws + 2 * n);
        auto go = [&](auto* kernel) {
          check_cuda(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                          (int)sizeof(unsigned) * kSortWarps * kBins),
                     "lookup_sort smem");
          launch_cluster(R, kernel, R + gather, kSortThreads, sizeof(unsigned) * kSortWarps << bits,
                         st, idx, (const T*)w, (T*)out, total, FastDiv(per), C, V, scale, n,
                         padding, passes, bits, passes & 1 ? a : b, passes & 1 ? b : a);
        };
        vec ? go(lookup_sort_kernel<T, true>) : go(lookup_sort_kernel<T, false>);
        if (!alone) continue;
      }
      auto go = [&](auto* kernel) {
        launch(kernel, grid_for(total, 256, kNumSMs * 16), 256, 0, st, idx + i, (const T*)w,
               (T*)out + i * C, total, FastDiv(per), C, V, scale);
      };
      vec ? go(lookup_kernel<T, true>) : go(lookup_kernel<T, false>);
    }
  });
  MSB_CHECK_LAUNCH("scaled_embedding_fwd");
}

// a flag a chunk, then the parts, 16-byte aligned
static long long flag_words(long long chunks) { return (chunks + 15) / 16 * 4; }
long long scaled_embedding_ws(long long n, int C) {
  const long long chunks = chunks_of(n);
  return flag_words(chunks) + chunks * 2 * C;
}

void scaled_embedding_bwd(const void* dout, const unsigned* sorted, void* grad, bool accumulate,
                          unsigned* ws, long long n, int C, long long V, float scale, int dtype,
                          cudaStream_t st) {
  const uint2* list = (const uint2*)sorted;
  const int slabs = (C + 255) / 256;
  const long long chunks = chunks_of(n);
  unsigned char* open = (unsigned char*)ws;
  float* part = (float*)(ws + flag_words(chunks));
  MSB_DISPATCH_FLOAT(dtype, T, {
    const bool vec = C % 8 == 0 && aligned16(dout) && aligned16(grad);
    const long long tasks = chunks * slabs;
    const unsigned row_blocks = (unsigned)((tasks + 7) / 8);
    // units to clear of 16 to 256 KB, eight a SM where the table allows: a unit
    // costs a search in the list
    const long long row = (long long)C * sizeof(T), even = V * row / (8 * kNumSMs);
    const long long fit = std::min(std::max(even, 16LL << 10), 256LL << 10) / row;
    const int unit = (int)(fit < 1 ? 1 : fit > kUnitRows ? kUnitRows : fit);
    const unsigned units = accumulate ? 0 : (unsigned)((V + unit - 1) / unit);
    auto rows = [&](auto* kernel) {
      if (row_blocks + units > 0)
        launch(kernel, row_blocks + units, 256, 0, st, list, n, (unsigned)V, (const T*)dout, C,
               FastDiv(slabs), (unsigned)tasks, (T*)grad, scale, part, open, row_blocks, unit);
    };
    auto runs = [&](auto* kernel) {
      const int cols = (C + kRunCols - 1) / kRunCols;
      if (chunks > 1)
        launch(kernel, (unsigned)((chunks + 31) / 32 * cols), kRunThreads, 0, st, list, n, part, C,
               chunks, FastDiv(cols), (T*)grad, scale, open);
    };
    auto go = [&](auto add) {
      constexpr bool A = decltype(add)::value;
      vec ? rows(sorted_rows_kernel<T, true, A>) : rows(sorted_rows_kernel<T, false, A>);
      C % 4 == 0 ? runs(sorted_runs_kernel<T, A, true>) : runs(sorted_runs_kernel<T, A, false>);
    };
    accumulate ? go(std::true_type{}) : go(std::false_type{});
  });
  MSB_CHECK_LAUNCH("scaled_embedding_bwd");
}

}  // namespace msb
