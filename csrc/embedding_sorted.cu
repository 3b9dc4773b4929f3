// Embedding lookup with scaling, and its gradient by sorted tokens.
//
//   out[i] = scale * W[idx_i]        dW[v] = scale * sum over {i : idx_i = v} of dout[i]
//
// The sum of a row is taken in fp32 in an order that depends on idx alone:
// the positions are sorted by token (stable, so ascending within a token), the
// sorted list is cut into chunks of 8 or 32 entries, and every run of one token is
// summed front to back inside a chunk; a run that crosses chunks leaves one
// fp32 partial per chunk, added up in chunk order.  No atomics touch values,
// so the gradient is the same from run to run, and no [V, C] accumulator is
// kept.
//
// Tokens outside [0, V) read as a zero row; they and the padding token get no
// gradient (key V, sorted behind all others).
#include <cooperative_groups.h>

#include "common.cuh"
#include "vec.cuh"

namespace msb {

MSB_BOUNDS_TU(embedding)

namespace {

namespace cg = cooperative_groups;

constexpr int kSortThreads = 1024;
constexpr int kDigit = 9;           // most bits of a sorting pass
constexpr int kBins = 1 << kDigit;
constexpr int kSortWarps = kSortThreads / 32;
constexpr int kMaxCluster = 8;
constexpr int kHeld = 4;            // entries a lane keeps in registers over a pass
constexpr int kRows = 8;            // rows in flight in the sum kernel

// VEC: eight columns a thread (width a multiple of 8, 16-byte aligned table)
template <typename T, bool VEC>
__global__ void __launch_bounds__(256)
scaled_embedding_fwd_kernel(const long long* __restrict__ idx, const T* __restrict__ w,
                            T* __restrict__ out, unsigned total, FastDiv per, int C, long long V,
                            float scale) {
  ::msb::pdl_begin();
  for (unsigned i = blockIdx.x * blockDim.x + threadIdx.x; i < total;
       i += gridDim.x * blockDim.x) {
    const unsigned m = per.div(i);
    const int c = (int)(i - m * per.d) * (VEC ? 8 : 1);
    const long long t = idx[m];
    const bool in = t >= 0 && t < V;
    if (c == 0) (void)MSB_OK(in, kSiteEmbeddingToken, t, V);
    if (VEC) {
      float f[8] = {0, 0, 0, 0, 0, 0, 0, 0};
      if (in) load8(w + t * C + c, f);
#pragma unroll
      for (int k = 0; k < 8; ++k) f[k] *= scale;
      store8(out + (long long)m * C + c, f);
    } else {
      out[(long long)m * C + c] = from_f32<T>(in ? to_f32(w[t * C + c]) * scale : 0.f);
    }
  }
}

// The first cluster sorts (token, position) by token, 9 bits or fewer a pass;
// the others meanwhile clear the gradient (fill_n vectors of 16 bytes, and
// fill_tail bytes behind them), where it is a new one.
//
// Every warp of the cluster owns one contiguous piece of the list.  A pass
// counts the digits of each warp's piece, turns the counts into places (over
// the warps of a block, over the blocks through distributed shared memory, over
// the digits), and writes each entry to its place, warp by warp in order, lanes
// with the same digit ranked by __match_any_sync: stable by construction.  The
// cluster barrier orders the passes.  What bounds it is the latency of its
// steps, not their work: 16384 tokens of 50257 take SORT16K us.
__global__ void __launch_bounds__(kSortThreads)
sort_tokens_kernel(const long long* __restrict__ idx, long long n, long long V,
                   long long padding, int passes, int bits, unsigned* key_a, unsigned* pos_a,
                   unsigned* key_b, unsigned* pos_b, uint4* fill, long long fill_n,
                   int fill_tail) {
  ::msb::pdl_begin();
  extern __shared__ unsigned cnt[];   // [kSortWarps][1 << bits]
  __shared__ unsigned hist[kBins], base[kBins], wsum[kSortWarps];
  cg::cluster_group cluster = cg::this_cluster();
  const unsigned q = cluster.block_rank(), R = cluster.num_blocks();
  if (blockIdx.x >= R) {
    const long long threads = (long long)(gridDim.x - R) * kSortThreads;
    const long long first = (long long)(blockIdx.x - R) * kSortThreads + threadIdx.x;
    for (long long i = first; i < fill_n; i += threads) fill[i] = make_uint4(0, 0, 0, 0);
    if (first < fill_tail) reinterpret_cast<unsigned char*>(fill + fill_n)[first] = 0;
    return;
  }
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int bins = 1 << bits;
  const unsigned ones = (unsigned)bins - 1u, below = (1u << lane) - 1u;
  const long long per = (n + (long long)R * kSortThreads - 1) / ((long long)R * kSortThreads) * 32;
  const long long lo = min(n, per * (q * kSortWarps + warp)), hi = min(n, lo + per);
  unsigned* mine = cnt + warp * bins;
  // entry i of a pass; behind the piece: a digit of its own, so that lanes match
  auto load = [&](int p, long long i, unsigned& key, unsigned& pos) {
    key = pos = 0;
    if (i >= hi) return;
    if (p == 0) {
      const long long t = idx[i];
      const bool in = t >= 0 && t < V;
      key = in && t != padding ? (unsigned)t : (unsigned)V;
      pos = (unsigned)i;
    } else {   // written by other blocks of the cluster
      key = __ldcg((p & 1 ? key_a : key_b) + i);
      pos = __ldcg((p & 1 ? pos_a : pos_b) + i);
    }
  };
  for (int p = 0; p < passes; ++p) {
    const int shift = p * bits;
    unsigned key[kHeld], pos[kHeld], same[kHeld];
#pragma unroll
    for (int h = 0; h < kHeld; ++h) load(p, lo + h * 32 + lane, key[h], pos[h]);
    for (int b = lane * 4; b < bins; b += 128)
      *reinterpret_cast<uint4*>(mine + b) = make_uint4(0, 0, 0, 0);
    __syncwarp();
    auto match = [&](unsigned k, long long i) {
      return __match_any_sync(0xffffffffu, i < hi ? (k >> shift) & ones : kBins);
    };
    auto count = [&](unsigned k, long long i, unsigned m) {
      if (i < hi && (m & below) == 0) mine[(k >> shift) & ones] += __popc(m);
      __syncwarp();
    };
#pragma unroll
    for (int h = 0; h < kHeld; ++h) {
      if (lo + h * 32 < hi) {
        same[h] = match(key[h], lo + h * 32 + lane);
        count(key[h], lo + h * 32 + lane, same[h]);
      }
    }
    for (long long i0 = lo + kHeld * 32; i0 < hi; i0 += 32) {
      unsigned k, at;
      load(p, i0 + lane, k, at);
      count(k, i0 + lane, match(k, i0 + lane));
    }
    __syncthreads();
    if (threadIdx.x < bins) {
      unsigned run = 0;
#pragma unroll
      for (int w = 0; w < kSortWarps; ++w) {
        const unsigned v = cnt[w * bins + threadIdx.x];
        cnt[w * bins + threadIdx.x] = run;
        run += v;
      }
      hist[threadIdx.x] = run;
    }
    cluster.sync();
    unsigned before = 0, all = 0;
    if (threadIdx.x < bins) {
      unsigned v[kMaxCluster];
#pragma unroll
      for (unsigned r = 0; r < kMaxCluster; ++r)
        v[r] = r < R ? *cluster.map_shared_rank(hist + threadIdx.x, r) : 0u;
#pragma unroll
      for (unsigned r = 0; r < kMaxCluster; ++r) {
        before += r < q ? v[r] : 0u;
        all += v[r];
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
    unsigned* key_out = p & 1 ? key_b : key_a;
    unsigned* pos_out = p & 1 ? pos_b : pos_a;
    auto place = [&](unsigned k, unsigned from, long long i, unsigned m) {
      const unsigned d = (k >> shift) & ones;
      if (i < hi) {
        const unsigned at = base[d] + mine[d] + __popc(m & below);
        key_out[at] = k;
        pos_out[at] = from;
      }
      __syncwarp();
      if (i < hi && (m & below) == 0) mine[d] += __popc(m);
      __syncwarp();
    };
#pragma unroll
    for (int h = 0; h < kHeld; ++h) {
      if (lo + h * 32 < hi) place(key[h], pos[h], lo + h * 32 + lane, same[h]);
    }
    for (long long i0 = lo + kHeld * 32; i0 < hi; i0 += 32) {
      unsigned k, from;
      load(p, i0 + lane, k, from);
      place(k, from, i0 + lane, match(k, i0 + lane));
    }
    cluster.sync();   // the list is written, and hist may be again
  }
}

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
      if (c0 < C) store8(row + c0, f);
    }
  }
};

// A warp sums a chunk of CHUNK sorted entries over 256 columns.  The rows of
// eight entries, and the gradient rows that their sums are added to, are loaded
// before any is used, whatever runs they belong to: most runs are one or two
// entries long, and run by run the loads would wait for one another.
template <typename T, bool VEC, bool ADD, int CHUNK>
__global__ void __launch_bounds__(256)
sorted_rows_kernel(const unsigned* __restrict__ keys, const unsigned* __restrict__ pos,
                   long long n, unsigned V, const T* __restrict__ dout, int C, FastDiv slabs,
                   unsigned tasks, T* grad, float scale, float* __restrict__ part) {
  ::msb::pdl_begin();
  const int lane = threadIdx.x & 31;
  const unsigned task = blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
  if (task >= tasks) return;
  const unsigned j = slabs.div(task);
  const long long first = (long long)j * CHUNK;
  const int c0 = (int)(task - j * slabs.d) * 256 + (VEC ? lane * 8 : lane);
  const int len = (int)min((long long)CHUNK, n - first);
  // lane l: entry l's token; what comes before and behind the chunk
  const unsigned my_key = lane < len ? keys[first + lane] : V;
  const unsigned my_pos = lane < len ? pos[first + lane] : 0u;
  const unsigned prev = first > 0 ? keys[first - 1] : V;
  const unsigned next = first + CHUNK < n ? keys[first + CHUNK] : V;
  unsigned behind = __shfl_down_sync(0xffffffffu, my_key, 1);   // the key after each entry
  if (lane == CHUNK - 1) behind = next;
  // entries that are tokens, and those that end a run inside the chunk
  const unsigned live = __ballot_sync(0xffffffffu, lane < len && my_key < V);
  const unsigned ends = __ballot_sync(0xffffffffu, lane < len && my_key < V && behind != my_key);
  if (live == 0) return;
  const unsigned key0 = __shfl_sync(0xffffffffu, my_key, 0);
  const int head = prev == key0 ? __ffs(~__ballot_sync(0xffffffffu, my_key == key0)) - 1 : 0;
  // `head` entries, when not 0, continue the run of the chunk before (32 of 32: -1)
  const unsigned in_head = prev != key0 ? 0u : head < 0 ? ~0u : (1u << head) - 1u;
  float a[8] = {0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll 1
  for (int e0 = 0; e0 < CHUNK; e0 += kRows) {
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
        float* d = part + ((long long)j * 2 + (in_head >> e & 1 ? 0 : 1)) * C;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int c = VEC ? c0 + i : c0 + 32 * i;
          if (c < C) d[c] = a[i];
        }
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) a[i] = 0.f;
    }
  }
}

// Block j adds up the run that begins in chunk j and goes on behind it: its
// threads look for the end together, then eight groups of warps add the parts
// of an eighth of the chunks each, and the eight sums are added in order.
constexpr int kRunThreads = 256;
constexpr int kRunGroups = 8;
template <typename T, bool ADD, int CHUNK>
__global__ void __launch_bounds__(kRunThreads)
sorted_runs_kernel(const unsigned* __restrict__ keys, long long n, unsigned V,
                   const float* __restrict__ part, int C, T* grad, float scale) {
  ::msb::pdl_begin();
  __shared__ float sums[kRunGroups][128];
  const long long j = blockIdx.x, first = j * CHUNK, after = first + CHUNK;
  if (after >= n) return;
  const unsigned key = keys[after];
  if (key >= V || keys[after - 1] != key) return;          // nothing goes on
  if (keys[first] == key && j > 0 && keys[first - 1] == key) return;   // began earlier
  long long count = 1;   // chunks that begin with this token, from j + 1 on
  for (;;) {
    const long long at = (j + 1 + count + threadIdx.x) * CHUNK;
    const int more = __syncthreads_count(at < n && keys[at] == key);
    count += more;
    if (more < kRunThreads) break;
  }
  T* g = grad + (long long)key * C;
  const float* p0 = part + (j * 2 + 1) * C;
  const float* p1 = part + (j + 1) * 2 * C;
  if (count <= 2 * kRunGroups) {   // few parts: a thread a column
    for (int c = threadIdx.x; c < C; c += kRunThreads) {
      float a = p0[c];
#pragma unroll 4
      for (int i = 0; i < (int)count; ++i) a += p1[(long long)i * 2 * C + c];
      g[c] = from_f32<T>(fmaf(a, scale, ADD ? to_f32(g[c]) : 0.f));
    }
    return;
  }
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const long long each = (count + kRunGroups - 1) / kRunGroups;
  const long long i0 = min(count, each * warp), i1 = min(count, i0 + each);
  for (int c0 = 0; c0 < C; c0 += 128) {
    float a[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (long long i = i0; i < i1; ++i) {
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int c = c0 + lane + 32 * k;
        if (c < C) a[k] += p1[i * 2 * C + c];
      }
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 4; ++k) sums[warp][lane + 32 * k] = a[k];
    __syncthreads();
    const int c = c0 + threadIdx.x;
    if (threadIdx.x < 128 && c < C) {
      float s = p0[c];
#pragma unroll
      for (int w = 0; w < kRunGroups; ++w) s += sums[w][threadIdx.x];
      g[c] = from_f32<T>(fmaf(s, scale, ADD ? to_f32(g[c]) : 0.f));
    }
  }
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// Entries of a chunk: 8 while that makes no more than 2^18 tasks (the more warps,
// the shorter their chains of loads), then 32 (fewer parts of cut runs).
int chunk_of(long long n, int slabs) { return n * slabs <= (8LL << 18) ? 8 : 32; }

}  // namespace

void scaled_embedding_fwd(const long long* idx, const void* w, void* out, long long n, int C,
                          long long V, float scale, int dtype, cudaStream_t st) {
  MSB_DISPATCH_FLOAT(dtype, T, {
    const bool vec = C % 8 == 0 && aligned16(w);
    const int per = vec ? C / 8 : C;
    const long long fit = (1LL << 30) / per, most = fit > 0 ? fit : 1;   // tokens a launch
    for (long long i = 0; i < n; i += most) {
      const unsigned total = (unsigned)((n - i < most ? n - i : most) * per);
      auto go = [&](auto* kernel) {
        launch(kernel, grid_for(total, 256, kNumSMs * 16), 256, 0, st, idx + i, (const T*)w,
               (T*)out + i * C, total, FastDiv(per), C, V, scale);
      };
      vec ? go(scaled_embedding_fwd_kernel<T, true>) : go(scaled_embedding_fwd_kernel<T, false>);
    }
  });
  MSB_CHECK_LAUNCH("scaled_embedding_fwd");
}

long long scaled_embedding_ws(long long n, int C) {
  const int chunk = chunk_of(n, (C + 255) / 256);
  return 4 * n + (n + chunk - 1) / chunk * 2 * C;
}

void scaled_embedding_bwd(const void* dout, const long long* idx, void* grad, bool accumulate,
                          unsigned* ws, long long n, int C, long long V, long long padding,
                          float scale, int dtype, cudaStream_t st) {
  // tokens and V itself (no token) in as few passes of at most kDigit bits
  int total_bits = 1;
  while ((V >> total_bits) != 0) ++total_bits;
  const int passes = n > 0 ? (total_bits + kDigit - 1) / kDigit : 0;
  // at least 2: a warp's counters are then whole vectors
  const int bits = passes > 0 && total_bits > 2 ? (total_bits + passes - 1) / passes : 2;
  unsigned *ka = ws, *pa = ws + n, *kb = ws + 2 * n, *pb = ws + 3 * n;
  float* part = reinterpret_cast<float*>(ws + 4 * n);
  unsigned R = 1;
  while (R < kMaxCluster && (long long)R * kSortThreads < n) R *= 2;
  const size_t smem = sizeof(unsigned) * kSortWarps << bits;
  check_cuda(cudaFuncSetAttribute(sort_tokens_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                  (int)(sizeof(unsigned) * kSortWarps * kBins)), "sort_tokens smem");
  const long long bytes = accumulate ? 0 : V * C * (dtype == kF32 ? 4 : 2);
  // the clearing blocks: 16 vectors a thread, in whole clusters
  const long long fill_n = bytes / 16;
  const long long blocks = (fill_n + 16 * kSortThreads - 1) / (16 * kSortThreads) + (bytes % 16 != 0);
  const unsigned extra = (unsigned)((blocks + R - 1) / R * R);
  if (n == 0 && extra == 0) return;
  launch_cluster(R, sort_tokens_kernel, R + extra, kSortThreads, smem, st, idx, n, V, padding,
                 passes, bits, ka, pa, kb, pb, (uint4*)grad, fill_n, (int)(bytes % 16));
  if (n == 0) return;
  const unsigned* keys = passes & 1 ? ka : kb;
  const unsigned* pos = passes & 1 ? pa : pb;
  const int slabs = (C + 255) / 256, chunk = chunk_of(n, slabs);
  const long long chunks = (n + chunk - 1) / chunk;
  MSB_DISPATCH_FLOAT(dtype, T, {
    const bool vec = C % 8 == 0 && aligned16(dout) && aligned16(grad);
    const long long tasks = chunks * slabs;
    auto rows = [&](auto* kernel) {
      launch(kernel, (unsigned)((tasks + 7) / 8), 256, 0, st, keys, pos, n, (unsigned)V,
             (const T*)dout, C, FastDiv(slabs), (unsigned)tasks, (T*)grad, scale, part);
    };
    auto runs = [&](auto* kernel) {
      if (chunks > 1)
        launch(kernel, (unsigned)chunks, kRunThreads, 0, st, keys, n, (unsigned)V, part, C,
               (T*)grad, scale);
    };
    if (chunk == 8) {
      if (accumulate) {
        vec ? rows(sorted_rows_kernel<T, true, true, 8>) : rows(sorted_rows_kernel<T, false, true, 8>);
        runs(sorted_runs_kernel<T, true, 8>);
      } else {
        vec ? rows(sorted_rows_kernel<T, true, false, 8>) : rows(sorted_rows_kernel<T, false, false, 8>);
        runs(sorted_runs_kernel<T, false, 8>);
      }
    } else {
      if (accumulate) {
        vec ? rows(sorted_rows_kernel<T, true, true, 32>) : rows(sorted_rows_kernel<T, false, true, 32>);
        runs(sorted_runs_kernel<T, true, 32>);
      } else {
        vec ? rows(sorted_rows_kernel<T, true, false, 32>) : rows(sorted_rows_kernel<T, false, false, 32>);
        runs(sorted_runs_kernel<T, false, 32>);
      }
    }
  });
  MSB_CHECK_LAUNCH("scaled_embedding_bwd");
}

}  // namespace msb
