// Embedding lookup with scaling, and its gradient by sorted tokens.
//
//   out[i] = scale * W[idx_i]        dW[v] = scale * sum over {i : idx_i = v} of dout[i]
//
// The sum of a row is taken in fp32 in an order that depends on idx alone:
// the positions are sorted by token (stable, so ascending within a token), the
// sorted list is cut into chunks of 32 entries, and every run of one token is
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

constexpr int kChunk = 32;          // sorted entries a warp sums
constexpr int kSortThreads = 1024;
constexpr int kDigit = 9;           // most bits of a sorting pass
constexpr int kBins = 1 << kDigit;
constexpr int kSortWarps = kSortThreads / 32;

template <typename T, bool VEC>
__global__ void __launch_bounds__(256)
scaled_embedding_fwd_kernel(const long long* __restrict__ idx, const T* __restrict__ w,
                            T* __restrict__ out, long long n, int C, long long V, float scale) {
  ::msb::pdl_begin();
  const int step = VEC ? 8 : 1;
  const int per = C / step;
  const long long total = n * per;
  for (long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x; i < total;
       i += (long long)gridDim.x * blockDim.x) {
    const long long m = i / per;
    const int c = (int)(i - m * per) * step;
    const long long t = idx[m];
    const bool in = t >= 0 && t < V;
    if (c == 0) (void)MSB_OK(in, kSiteEmbeddingToken, t, V);
    if (VEC) {
      float f[8] = {0, 0, 0, 0, 0, 0, 0, 0};
      if (in) load8(w + t * C + c, f);
#pragma unroll
      for (int k = 0; k < 8; ++k) f[k] *= scale;
      store8(out + m * C + c, f);
    } else {
      out[m * C + c] = from_f32<T>(in ? to_f32(w[t * C + c]) * scale : 0.f);
    }
  }
}

// One cluster sorts (token, position) by token, 9 bits or fewer a pass.  Every
// warp of the cluster owns one contiguous piece of the list.  A pass counts
// the digits of each warp's piece, turns the counts into places (over the
// warps of a block, over the blocks through distributed shared memory, over
// the digits), and writes each entry to its place, warp by warp in order,
// lanes with the same digit ranked by __match_any_sync: stable by
// construction.  The cluster barrier orders the passes.
__global__ void __launch_bounds__(kSortThreads)
sort_tokens_kernel(const long long* __restrict__ idx, long long n, long long V,
                   long long padding, int passes, int bits, unsigned* key_a, unsigned* pos_a,
                   unsigned* key_b, unsigned* pos_b) {
  ::msb::pdl_begin();
  extern __shared__ unsigned cnt[];   // [kSortWarps][kBins]
  __shared__ unsigned hist[kBins], base[kBins], wsum[kSortWarps];
  cg::cluster_group cluster = cg::this_cluster();
  const unsigned q = cluster.block_rank(), R = cluster.num_blocks();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const long long per = (n + (long long)R * kSortThreads - 1) / ((long long)R * kSortThreads) * 32;
  const long long lo = min(n, per * (q * kSortWarps + warp)), hi = min(n, lo + per);
  const unsigned ones = (1u << bits) - 1u;
  unsigned* mine = cnt + warp * kBins;
  auto load = [&](int p, long long i, unsigned& key, unsigned& pos) {
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
    for (int b = lane; b < kBins; b += 32) mine[b] = 0;
    __syncwarp();
    for (long long i = lo + lane; i < hi; i += 32) {
      unsigned key, pos;
      load(p, i, key, pos);
      atomicAdd(mine + ((key >> shift) & ones), 1u);
    }
    __syncthreads();
    if (threadIdx.x < kBins) {
      unsigned run = 0;
#pragma unroll 8
      for (int w = 0; w < kSortWarps; ++w) {
        const unsigned v = cnt[w * kBins + threadIdx.x];
        cnt[w * kBins + threadIdx.x] = run;
        run += v;
      }
      hist[threadIdx.x] = run;
    }
    cluster.sync();
    unsigned before = 0, all = 0;
    if (threadIdx.x < kBins) {
      for (unsigned r = 0; r < R; ++r) {
        const unsigned v = *cluster.map_shared_rank(hist + threadIdx.x, r);
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
    if (threadIdx.x < kBins) {
      unsigned lower = 0;
      for (int w = 0; w < warp; ++w) lower += wsum[w];
      base[threadIdx.x] = lower + incl - all + before;
    }
    __syncthreads();
    unsigned* key_out = p & 1 ? key_b : key_a;
    unsigned* pos_out = p & 1 ? pos_b : pos_a;
    for (long long i0 = lo; i0 < hi; i0 += 32) {
      const long long i = i0 + lane;
      const bool on = i < hi;
      unsigned key = 0, pos = 0;
      if (on) load(p, i, key, pos);
      const unsigned d = on ? (key >> shift) & ones : kBins;   // an idle lane matches idle lanes
      const unsigned same = __match_any_sync(0xffffffffu, d);
      if (on) {
        const unsigned at = base[d] + mine[d] + __popc(same & ((1u << lane) - 1u));
        key_out[at] = key;
        pos_out[at] = pos;
      }
      __syncwarp();
      if (on && lane == 31 - __clz(same)) mine[d] += __popc(same);
      __syncwarp();
    }
    cluster.sync();   // the list is written, and hist may be again
  }
}

// where a run of sorted entries [e0, e1) of chunk j is cut off
struct Run {
  bool left, right;   // goes on in the chunk before, after
};

template <typename T>
__device__ __forceinline__ void put8(T* p, const float (&a)[8], float scale, bool accumulate) {
  float o[8];
  if (accumulate) {
    load8(p, o);
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k) o[k] = 0.f;
  }
#pragma unroll
  for (int k = 0; k < 8; ++k) o[k] = fmaf(a[k], scale, o[k]);
  store8(p, o);
}

// A warp sums one chunk of the sorted list over 256 columns, 8 a lane (VEC:
// adjacent ones; otherwise 32 apart, for widths and addresses that do not
// allow 16-byte accesses).
template <typename T, bool VEC>
__global__ void __launch_bounds__(256)
sorted_rows_kernel(const unsigned* __restrict__ keys, const unsigned* __restrict__ pos,
                   long long n, unsigned V, const T* __restrict__ dout, int C, int slabs,
                   T* __restrict__ grad, float scale, bool accumulate,
                   float* __restrict__ part) {
  ::msb::pdl_begin();
  const int lane = threadIdx.x & 31;
  const long long task = (long long)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
  const long long j = task / slabs, first = j * kChunk;
  const int slab = (int)(task - j * slabs);
  if (first >= n) return;
  const int len = (int)min((long long)kChunk, n - first);
  const unsigned my_key = lane < len ? keys[first + lane] : V;
  const unsigned my_pos = lane < len ? pos[first + lane] : 0u;
  const unsigned prev = first > 0 ? keys[first - 1] : V;
  const unsigned next = first + kChunk < n ? keys[first + kChunk] : V;
  const int c0 = slab * 256 + (VEC ? lane * 8 : lane);
  auto load = [&](unsigned p, float (&f)[8]) {
    const T* row = dout + (long long)p * C;
    if (VEC) {
      if (c0 < C) load8(row + c0, f);
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k) f[k] = c0 + 32 * k < C ? to_f32(row[c0 + 32 * k]) : 0.f;
    }
  };
  int e = 0;
  while (e < len) {
    const unsigned key = __shfl_sync(0xffffffffu, my_key, e);
    if (key >= V) break;   // sorted behind all tokens
    const unsigned same = __ballot_sync(0xffffffffu, my_key == key && lane < len);
    const int end = e + __popc(same);
    float a[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    for (int i = e; i < end; i += 4) {
      float f[4][8];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const unsigned p = __shfl_sync(0xffffffffu, my_pos, min(i + u, 31));
#pragma unroll
        for (int k = 0; k < 8; ++k) f[u][k] = 0.f;
        if (i + u < end) load(p, f[u]);
      }
#pragma unroll
      for (int u = 0; u < 4; ++u)
#pragma unroll
        for (int k = 0; k < 8; ++k) a[k] += f[u][k];
    }
    const Run cut = {e == 0 && prev == key, end == kChunk && next == key};
    if (!cut.left && !cut.right) {
      T* g = grad + (long long)key * C;
      if (VEC) {
        if (c0 < C) put8(g + c0, a, scale, accumulate);
      } else {
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const int c = c0 + 32 * k;
          if (c < C) g[c] = from_f32<T>(fmaf(a[k], scale, accumulate ? to_f32(g[c]) : 0.f));
        }
      }
    } else {
      float* d = part + (j * 2 + (cut.left ? 0 : 1)) * C;
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const int c = VEC ? c0 + k : c0 + 32 * k;
        if (c < C) d[c] = a[k];
      }
    }
    e = end;
  }
}

// Block j adds up the run that begins in chunk j and goes on behind it.
template <typename T>
__global__ void __launch_bounds__(256)
sorted_runs_kernel(const unsigned* __restrict__ keys, long long n, unsigned V,
                   const float* __restrict__ part, int C, T* __restrict__ grad, float scale,
                   bool accumulate) {
  ::msb::pdl_begin();
  const long long j = blockIdx.x, first = j * kChunk, after = first + kChunk;
  if (after >= n) return;
  const unsigned key = keys[after];
  if (key >= V || keys[after - 1] != key) return;          // nothing goes on
  if (keys[first] == key && j > 0 && keys[first - 1] == key) return;   // began earlier
  long long last = j + 1;   // the last chunk that begins with this token
  while ((last + 1) * kChunk < n && keys[(last + 1) * kChunk] == key) ++last;
  T* g = grad + (long long)key * C;
  for (int c = threadIdx.x; c < C; c += blockDim.x) {
    float a = part[(j * 2 + 1) * C + c];
    for (long long i = j + 1; i <= last; ++i) a += part[i * 2 * C + c];
    g[c] = from_f32<T>(fmaf(a, scale, accumulate ? to_f32(g[c]) : 0.f));
  }
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

}  // namespace

void scaled_embedding_fwd(const long long* idx, const void* w, void* out, long long n, int C,
                          long long V, float scale, int dtype, cudaStream_t st) {
  if (n == 0) return;
  MSB_DISPATCH_FLOAT(dtype, T, {
    if (C % 8 == 0 && aligned16(w)) {
      launch(scaled_embedding_fwd_kernel<T, true>, grid_for(n * (C / 8), 256, kNumSMs * 16), 256,
             0, st, idx, (const T*)w, (T*)out, n, C, V, scale);
    } else {
      launch(scaled_embedding_fwd_kernel<T, false>, grid_for(n * C, 256, kNumSMs * 16), 256, 0,
             st, idx, (const T*)w, (T*)out, n, C, V, scale);
    }
  });
  MSB_CHECK_LAUNCH("scaled_embedding_fwd");
}

long long scaled_embedding_ws(long long n, int C) {
  return 4 * n + (n + kChunk - 1) / kChunk * 2 * C;
}

void scaled_embedding_bwd(const void* dout, const long long* idx, void* grad, bool accumulate,
                          unsigned* ws, long long n, int C, long long V, long long padding,
                          float scale, int dtype, cudaStream_t st) {
  if (n == 0) return;
  // tokens and V itself (no token) in as few passes of at most kDigit bits
  int total_bits = 1;
  while ((V >> total_bits) != 0) ++total_bits;
  const int passes = (total_bits + kDigit - 1) / kDigit;
  const int bits = (total_bits + passes - 1) / passes;
  unsigned *ka = ws, *pa = ws + n, *kb = ws + 2 * n, *pb = ws + 3 * n;
  float* part = reinterpret_cast<float*>(ws + 4 * n);
  unsigned R = 1;
  while (R < 8 && (long long)R * kSortThreads < n) R *= 2;
  const size_t smem = sizeof(unsigned) * kSortWarps * kBins;
  check_cuda(cudaFuncSetAttribute(sort_tokens_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                  (int)smem), "sort_tokens smem");
  launch_cluster(R, sort_tokens_kernel, R, kSortThreads, smem, st, idx, n, V, padding, passes,
                 bits, ka, pa, kb, pb);
  const unsigned* keys = passes & 1 ? ka : kb;
  const unsigned* pos = passes & 1 ? pa : pb;
  const long long chunks = (n + kChunk - 1) / kChunk;
  const int slabs = (C + 255) / 256;
  MSB_DISPATCH_FLOAT(dtype, T, {
    const unsigned blocks = (unsigned)((chunks * slabs + 7) / 8);
    if (C % 8 == 0 && aligned16(dout) && aligned16(grad)) {
      launch(sorted_rows_kernel<T, true>, blocks, 256, 0, st, keys, pos, n, (unsigned)V,
             (const T*)dout, C, slabs, (T*)grad, scale, accumulate, part);
    } else {
      launch(sorted_rows_kernel<T, false>, blocks, 256, 0, st, keys, pos, n, (unsigned)V,
             (const T*)dout, C, slabs, (T*)grad, scale, accumulate, part);
    }
    if (chunks > 1) {
      launch(sorted_runs_kernel<T>, (unsigned)chunks, 256, 0, st, keys, n, (unsigned)V, part, C,
             (T*)grad, scale, accumulate);
    }
  });
  MSB_CHECK_LAUNCH("scaled_embedding_bwd");
}

}  // namespace msb
