// Log probabilities of given tokens, with the entropy of every position and
// its most probable alternatives, over model-dtype logits; and their gradient.
//
// Row x[0..V), temperature T, c = log2(e) / T, m = max(x), z_i = x_i c - m c:
//
//   s = sum 2^z_i      t = sum 2^z_i z_i
//   log p_i = ln 2 (z_i - log2 s)        H = ln 2 (log2 s - t / s)
//
// and for upstream gradients g_i of the log probabilities asked for (the token
// and the alternatives), G their sum, gH of the entropy,
//
//   dx_i = (g_i - p_i G - gH p_i (log p_i + H)) / T.
//
// A logit of -inf has probability zero and adds nothing anywhere; a row with
// nothing else is empty: its log probabilities are -inf, its entropy and its
// gradient zero.  A NaN or +inf in a row makes all its values NaN.
#include <cooperative_groups.h>

#include "common.cuh"
#include "vec.cuh"

namespace msb {

MSB_BOUNDS_TU(logprob)

namespace {

namespace cg = cooperative_groups;

constexpr int kThreads = 256;
constexpr int kMaxK = 32;
constexpr int kMaxCluster = 8;
constexpr int kGroups = 64;    // groups of threads whose maxima give a threshold, >= kMaxK
constexpr int kCand = 1024;    // candidates kept above the threshold, and
constexpr int kEqual = 512;    // at it
static_assert(kGroups * 4 == kThreads && kMaxK <= kGroups, "a group is four threads of a warp");
static_assert(kMaxK + kEqual <= kCand, "what is ranked fits");

// 16 bytes of logits
template <typename T>
struct Vec {
  static constexpr int N = 16 / sizeof(T);
  uint4 r;
  __device__ __forceinline__ void unpack(float (&f)[N]) const {
    if constexpr (sizeof(T) == 2) {
      unpack_u4<T>(r, f);
    } else {
      f[0] = __uint_as_float(r.x);
      f[1] = __uint_as_float(r.y);
      f[2] = __uint_as_float(r.z);
      f[3] = __uint_as_float(r.w);
    }
  }
  // the larger of this and another, place by place, two at a time in 16 bits; a
  // NaN only where both are
  __device__ __forceinline__ Vec larger(const Vec& o) const {
    Vec m;
    if constexpr (sizeof(T) == 2) {
      using T2 = std::conditional_t<std::is_same<T, __half>::value, __half2, __nv_bfloat162>;
      const T2 *p = reinterpret_cast<const T2*>(&r), *q = reinterpret_cast<const T2*>(&o.r);
#pragma unroll
      for (int i = 0; i < 4; ++i) reinterpret_cast<T2*>(&m.r)[i] = __hmax2(p[i], q[i]);
    } else {
      const float *p = reinterpret_cast<const float*>(&r), *q = reinterpret_cast<const float*>(&o.r);
#pragma unroll
      for (int i = 0; i < 4; ++i) reinterpret_cast<float*>(&m.r)[i] = fmaxf(p[i], q[i]);
    }
    return m;
  }
  // a load that stays where it stands in the program
  __device__ __forceinline__ void load(const uint4* p) {
    asm volatile("ld.global.nc.v4.u32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "l"(p));
  }
  // -inf everywhere
  __device__ __forceinline__ void clear() {
    const unsigned w = sizeof(T) == 4 ? 0xff800000u
                       : std::is_same<T, __half>::value ? 0xfc00fc00u : 0xff80ff80u;
    r = make_uint4(w, w, w, w);
  }
  // the largest value that is no NaN (a NaN where all are)
  __device__ __forceinline__ float max() const {
    if constexpr (std::is_same<T, __nv_bfloat16>::value) {
      const __nv_bfloat162* p = reinterpret_cast<const __nv_bfloat162*>(&r);
      const __nv_bfloat162 m = __hmax2(__hmax2(p[0], p[1]), __hmax2(p[2], p[3]));
      return fmaxf(__low2float(m), __high2float(m));
    } else if constexpr (std::is_same<T, __half>::value) {
      const __half2* p = reinterpret_cast<const __half2*>(&r);
      const __half2 m = __hmax2(__hmax2(p[0], p[1]), __hmax2(p[2], p[3]));
      return fmaxf(__low2float(m), __high2float(m));
    } else {
      return fmaxf(fmaxf(__uint_as_float(r.x), __uint_as_float(r.y)),
                   fmaxf(__uint_as_float(r.z), __uint_as_float(r.w)));
    }
  }
};

// (value, index) as one number: larger value first, then the lower index.
// NaN has no place in the order (0).
__device__ __forceinline__ unsigned order_of(float v) {
  const int b = __float_as_int(v + 0.f);  // -0 counts as 0
  return b < 0 ? ~(unsigned)b : (unsigned)b | 0x80000000u;
}
__device__ __forceinline__ float value_of(unsigned u) {
  return __int_as_float((int)(u & 0x80000000u ? u & 0x7fffffffu : ~u));
}
__device__ __forceinline__ unsigned long long key_of(float v, int i) {
  return v != v ? 0ull : ((unsigned long long)order_of(v) << 32) | (0xffffffffu - (unsigned)i);
}
__device__ __forceinline__ int key_index(unsigned long long k) {
  return (int)(0xffffffffu - (unsigned)k);
}

// The exponents of a row are z = x c - m c, one fused operation on the rounded
// product m c (the same one wherever the row's z are computed, so its rounding
// cancels).  That rounding shifts them by up to 2^-24 |m c|: where |m c| reaches
// 2^24 (a mask of -1e9 is not far from it, the lowest value of fp32 beyond fp32's
// range) the row is `wide` and z = (x - m) c.  A reference is held to that range, so
// a thread whose values all lie below it sums them relative to its lower end, next
// to which they still count; a block of a shared row whose own part is wide sums it
// relative to the part's maximum.
constexpr float kWide = 16777216.f;
__device__ __forceinline__ bool is_wide(float m, float c) {
  return fabsf(m * c) >= kWide && m != -INFINITY;
}
__device__ __forceinline__ float reference(float m, float c) {   // of -inf: 0
  return m == -INFINITY ? 0.f : fminf(fmaxf(m * c, -kWide), kWide);
}

// exponents at or under this give 2^z = 0; a larger one in z's place keeps
// 0 * z a number
constexpr float kLowZ = -200.f;

// A thread's maximum, and its sums relative to a reference that trails it: only
// a value more than 2^kSlack above moves it.  Some lane of a warp finds a new
// maximum in most vectors, so following it exactly would rescale in most.
constexpr float kSlack = 16.f;
struct Sums {
  float m = -INFINITY, ref = -1e37f;
  float2 s = {0.f, 0.f}, t = {0.f, 0.f};   // of even and odd values
  __device__ __forceinline__ void rebase(float to) {   // to a reference above
    const float d = fminf(fmaxf(ref - to, kLowZ), 0.f), f = ex2_approx(d);
    t = make_float2(f * fmaf(s.x, d, t.x), f * fmaf(s.y, d, t.y));
    s = make_float2(s.x * f, s.y * f);
    ref = to;
  }
  __device__ __forceinline__ void see(float v, float c) {
    m = fmaxf(m, v);
    if (fmaf(v, c, -ref) > kSlack) rebase(reference(v, c));
  }
};

template <bool ENT>
__device__ __forceinline__ void add_z(Sums& a, float2 z) {
  if (ENT) z = make_float2(max_nan(z.x, kLowZ), max_nan(z.y, kLowZ));
  const float2 e = make_float2(ex2_approx(z.x), ex2_approx(z.y));
  a.s = add2(a.s, e);
  if (ENT) a.t = fma2(e, z, a.t);
}

template <typename T, bool ENT>
__device__ __forceinline__ void add_vec(Sums& a, const Vec<T>& v, float c) {
  constexpr int N = Vec<T>::N;
  float x[N];
  v.unpack(x);
  const float2 c2 = make_float2(c, c), r2 = make_float2(-a.ref, -a.ref);
#pragma unroll
  for (int k = 0; k < N; k += 2) add_z<ENT>(a, fma2(make_float2(x[k], x[k + 1]), c2, r2));
}

template <bool ENT>
__device__ __forceinline__ void add_one(Sums& a, float x, float c) {
  a.see(x, c);
  add_z<ENT>(a, make_float2(fmaf(x, c, -a.ref), -INFINITY));
}

// The part of a row that a block of the cluster reads: vectors [v0, v1) of the
// row's aligned middle; the first block also has the `head` values before it,
// the last the `tail` behind it.
template <typename T>
struct Part {
  const T* row;
  const uint4* mid;
  int head, tail, nv, v0, v1, V;
  bool first, last;
  __device__ Part(const T* row_, int V_, unsigned q, unsigned R) : row(row_), V(V_) {
    constexpr int N = Vec<T>::N;
    const int off = (int)((16 - (reinterpret_cast<uintptr_t>(row) & 15)) & 15) / (int)sizeof(T);
    head = min(off, V);
    nv = (V - head) / N;
    tail = V - head - nv * N;
    mid = reinterpret_cast<const uint4*>(row + head);
    const int per = (nv + (int)R - 1) / (int)R;
    v0 = min(nv, per * (int)q);
    v1 = min(nv, v0 + per);
    first = q == 0;
    last = q == R - 1;
  }
  // index of a vector's first value
  __device__ __forceinline__ int at(int v) const { return head + v * Vec<T>::N; }
  // number of this block's values outside vectors, and the index of one
  __device__ __forceinline__ int loose() const { return (first ? head : 0) + (last ? tail : 0); }
  __device__ __forceinline__ int loose_at(int i) const {
    return first && i < head ? i : V - tail + i - (first ? head : 0);
  }
};

__device__ __forceinline__ float max_of_warp(float v) {   // v is no NaN
  float m;
  asm("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(m) : "f"(v));
  return m;
}

// A reduction over the block in two halves, so that several share one barrier.
template <typename F>
__device__ __forceinline__ void reduce_warps(float v, float* buf, F&& f) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = f(v, __shfl_xor_sync(0xffffffffu, v, o));
  if ((threadIdx.x & 31) == 0) buf[threadIdx.x >> 5] = v;
}
template <typename F>
__device__ __forceinline__ float reduce_block(const float* buf, F&& f) {   // after a barrier
  float v = buf[threadIdx.x & (kThreads / 32 - 1)];
#pragma unroll
  for (int o = kThreads / 64; o > 0; o >>= 1) v = f(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}

__device__ __forceinline__ void cluster_arrive() {
  asm volatile("barrier.cluster.arrive.release;" ::: "memory");
}
__device__ __forceinline__ void cluster_wait() {
  asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
}

// What the blocks of a row write into the first one's memory.
struct alignas(16) Joined {
  unsigned long long best[kMaxCluster * kMaxK];
  float m[kMaxCluster], s[kMaxCluster], t[kMaxCluster];
};
struct alignas(16) Top {
  unsigned long long best[kMaxK];      // its alternatives, best first; 0: none
  unsigned long long cand[kCand];
  unsigned long long equal[kEqual];
  unsigned long long round[kThreads / 32];
  unsigned group[kGroups];
  unsigned short winner[kThreads];
  float threshold;
  int winners, above, at;
};

// The k best of `n` keys in order, by counting for each how many beat it.
__device__ __forceinline__ void rank_keys(const unsigned long long* keys, int n,
                                          unsigned long long* out, int k) {
  for (int i = threadIdx.x; i < n; i += kThreads) {
    const unsigned long long mine = keys[i];
    if (mine == 0) continue;
    int r = 0, j = 0;
#pragma unroll 4
    for (; j + 2 <= n; j += 2) {
      const ulonglong2 two = *reinterpret_cast<const ulonglong2*>(keys + j);
      r += (two.x > mine) + (two.y > mine);
    }
    if (j < n) r += keys[j] > mine;
    if (r < k) out[r] = mine;
  }
}

// The block's k best values.  Every thread has the maximum of its values; the
// k-th largest of 64 maxima of four threads each is a threshold that at least k
// values reach and few exceed.  Only the values of the threads whose maximum
// reaches it are read again (from L2), the ones above the threshold collected
// and ranked.  Values equal to it are taken in index order: collected too or,
// where a row has very many (a mask), found by a scan from the front.
//
// Three steps with a barrier after each of the first two, which the kernel
// shares with its sums.
__device__ __forceinline__ void top_groups(float my_max, int k, Top& sh) {
  constexpr int A_WARP = kGroups / (kThreads / 32);
  const int tid = threadIdx.x, lane = tid & 31;
  float m = my_max;
#pragma unroll
  for (int o = A_WARP; o < 32; o <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  if (lane < A_WARP) sh.group[(tid >> 5) * A_WARP + lane] = order_of(m);
  if (tid < k) sh.best[tid] = 0;
  if (tid == 0) sh.winners = sh.above = sh.at = 0;
}
__device__ __forceinline__ void top_threshold(int k, Top& sh) {
  // four threads a group, each against a quarter of the groups
  const int g = threadIdx.x >> 2, part = threadIdx.x & 3;
  const unsigned mine = sh.group[g];
  int r = 0;
#pragma unroll
  for (int i = 0; i < kGroups / 16; ++i) {
    const int j = (i * 4 + part) * 4;
    const uint4 o = *reinterpret_cast<const uint4*>(sh.group + j);
    r += o.x > mine || (o.x == mine && j < g);
    r += o.y > mine || (o.y == mine && j + 1 < g);
    r += o.z > mine || (o.z == mine && j + 2 < g);
    r += o.w > mine || (o.w == mine && j + 3 < g);
  }
  r += __shfl_xor_sync(0xffffffffu, r, 1);
  r += __shfl_xor_sync(0xffffffffu, r, 2);
  if (r == k - 1 && part == 0) sh.threshold = value_of(mine);
}
template <typename T>
__device__ void top_of_part(const Part<T>& p, float my_max, int k, Top& sh) {
  constexpr int N = Vec<T>::N;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const float thr = sh.threshold;
  if (my_max >= thr) sh.winner[atomicAdd(&sh.winners, 1)] = (unsigned short)tid;
  __syncthreads();
  auto take = [&](float v, int i) {
    if (v > thr) {
      const int n = atomicAdd(&sh.above, 1);
      if (n < kCand) sh.cand[n] = key_of(v, i);
    } else if (v == thr) {
      const int n = atomicAdd(&sh.at, 1);
      if (n < kEqual) sh.equal[n] = key_of(v, i);
    }
  };
  // a warp a winner, a lane a vector of its
  const int winners = sh.winners;
  for (int w = warp; w < winners; w += kThreads / 32) {
    for (int v = p.v0 + sh.winner[w] + lane * kThreads; v < p.v1; v += 32 * kThreads) {
      Vec<T> x;
      x.r = p.mid[v];
      if (!(x.max() >= thr)) continue;
      float f[N];
      x.unpack(f);
#pragma unroll
      for (int j = 0; j < N; ++j) take(f[j], p.at(v) + j);
    }
  }
  for (int i = tid; i < p.loose(); i += kThreads) {
    const int at = p.loose_at(i);
    take(to_f32(p.row[at]), at);
  }
  __syncthreads();
  const int above = sh.above, equal = sh.at;
  if (above <= kCand) {
    const int need = min(k - above, equal);
    if (need > 0 && equal <= kEqual) {   // above < k <= kMaxK: there is room
      for (int i = tid; i < equal; i += kThreads) sh.cand[above + i] = sh.equal[i];
      __syncthreads();
      rank_keys(sh.cand, above + equal, sh.best, k);
      __syncthreads();
      return;
    }
    // the strictly larger ones, then the first `need` equal ones
    rank_keys(sh.cand, above, sh.best, k);
    if (need > 0 && warp == 0) {
      int found = 0;
      auto put = [&](bool is, int i) {   // lanes hold ascending indexes
        const unsigned b = __ballot_sync(0xffffffffu, is);
        const int r = found + __popc(b & ((1u << lane) - 1u));
        if (is && r < need) sh.best[above + r] = key_of(thr, i);
        found += __popc(b);
      };
      if (p.first) put(lane < p.head && to_f32(p.row[min(lane, p.V - 1)]) == thr, lane);
      const int e0 = p.at(p.v0), e1 = p.at(p.v1);
      for (int i = e0; i < e1 && found < need; i += 32) {
        const bool in = i + lane < e1;
        put(in && to_f32(p.row[in ? i + lane : e0]) == thr, i + lane);
      }
      if (p.last && found < need) {
        const int i = p.V - p.tail + lane;
        put(i < p.V && to_f32(p.row[min(i, p.V - 1)]) == thr, i);
      }
    }
    __syncthreads();
    return;
  }
  // more values above the threshold than are kept: the best one k times
  unsigned long long last = ~0ull;
  for (int j = 0; j < k; ++j) {
    unsigned long long b = 0;
    auto see = [&](int i) {
      const unsigned long long q = key_of(to_f32(p.row[i]), i);
      if (q < last && q > b) b = q;
    };
    for (int i = p.at(p.v0) + tid; i < p.at(p.v1); i += kThreads) see(i);
    for (int i = tid; i < p.loose(); i += kThreads) see(p.loose_at(i));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const unsigned long long w = __shfl_xor_sync(0xffffffffu, b, o);
      b = w > b ? w : b;
    }
    __syncthreads();
    if (lane == 0) sh.round[warp] = b;
    __syncthreads();
    b = sh.round[0];
    for (int w = 1; w < kThreads / 32; ++w) b = sh.round[w] > b ? sh.round[w] : b;
    last = b;
    if (tid == 0) sh.best[j] = b;
  }
  __syncthreads();
}

// A block a row or, SPLIT, a cluster a row where rows are few: then a thread has
// twice the vectors in flight, as it has few in all; in fp32 as well, where a
// vector is half the work (1021 x 32003: 29 us, 33 with four and more blocks).
//
// Bound in 16 bits by DRAM: 8192 x 50257 fp16, a tenth of it ignored, 119 us (6.2
// TB/s, 0.95 of the copy rate; XU pipe 75%, issue slots 56%), with the entropy 125,
// with 8 alternatives 139; 2048 x 128256 bf16 90, 92, 109.  The alternatives add
// their second look and its barriers, when nothing is at its limit (DRAM 0.85 of the
// copy rate, XU pipe 60%, issue slots 59%).
template <typename T, bool ENT, bool TOP, bool SPLIT>
__global__ void __launch_bounds__(kThreads, SPLIT ? 3 : sizeof(T) == 4 ? 4 : 6)
logprob_fwd_kernel(const T* __restrict__ logits, long long ld, const long long* __restrict__ tok,
                   int V, float c, float inv_t, long long ignore_index, int k,
                   float* __restrict__ logp, float* __restrict__ entropy,
                   float* __restrict__ top_logp, long long* __restrict__ top_tok,
                   float* __restrict__ stats) {
  ::msb::pdl_begin();
  __shared__ float buf[3][kThreads / 32];
  __shared__ std::conditional_t<TOP, Top, int> top;
  __shared__ std::conditional_t<SPLIT, Joined, int> joined;
  cg::cluster_group cluster = cg::this_cluster();
  const unsigned R = SPLIT ? cluster.num_blocks() : 1, q = SPLIT ? cluster.block_rank() : 0;
  const long long r = blockIdx.x / R;
  const T* row = logits + r * ld;
  const int tid = threadIdx.x;
  const Part<T> p(row, V, q, R);
  constexpr int U = SPLIT || sizeof(T) == 4 ? 8 : 4;   // vectors in flight a thread
  Vec<T> x[U];
  auto load = [&](int v) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      x[u].clear();
      if (v + u * kThreads >= p.v1) continue;
      if constexpr (SPLIT) {
        x[u].load(p.mid + v + u * kThreads);
      } else {
        x[u].r = p.mid[v + u * kThreads];
      }
    }
  };
  if constexpr (SPLIT) {
    load(p.v0 + tid);   // on its way while the token is
    cluster_arrive();   // waited for before the first block's memory is written
  }
  const long long t = tok[r];
  if (t == ignore_index) {   // in all blocks of the cluster alike
    if (q == 0 && tid == 0) {
      logp[r] = 0.f;
      if (ENT) entropy[r] = 0.f;
    }
    if (TOP && q == 0 && tid < k) {
      top_logp[r * k + tid] = 0.f;
      top_tok[r * k + tid] = -1;
    }
    return;
  }
  const bool in = t >= 0 && t < V;
  const float xt = q == 0 && tid == 0 && in ? to_f32(row[t]) : 0.f;

  Sums a;
  for (int v = p.v0 + tid; v < p.v1; v += U * kThreads) {
    if (!SPLIT || v != p.v0 + tid) load(v);
    Vec<T> top_of = x[0];
#pragma unroll
    for (int u = 1; u < U; ++u) top_of = top_of.larger(x[u]);
    a.see(top_of.max(), c);
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (v + u * kThreads < p.v1) add_vec<T, ENT>(a, x[u], c);
  }
  if (tid < p.loose()) add_one<ENT>(a, to_f32(row[p.loose_at(tid)]), c);
  const float my_max = a.m;

  auto larger = [](float x, float y) { return fmaxf(x, y); };
  auto sum = [](float x, float y) { return x + y; };
  const float warp_max = max_of_warp(my_max);
  if ((tid & 31) == 0) buf[0][tid >> 5] = warp_max;
  if constexpr (TOP) top_groups(my_max, k, top);
  __syncthreads();
  float m = reduce_block(buf[0], larger);   // of the block's part
  bool wide = is_wide(m, c);
  float ref = reference(m, c);
  if (wide && m != INFINITY) {   // once more, with differences
    a.s = a.t = make_float2(0.f, 0.f);
    for (int i = p.at(p.v0) + tid; i < p.at(p.v1); i += kThreads)
      add_z<ENT>(a, make_float2((to_f32(row[i]) - m) * c, -INFINITY));
    for (int i = tid; i < p.loose(); i += kThreads)
      add_z<ENT>(a, make_float2((to_f32(row[p.loose_at(i)]) - m) * c, -INFINITY));
  } else {
    a.rebase(ref);
  }
  reduce_warps(a.s.x + a.s.y, buf[1], sum);
  if (ENT) reduce_warps(a.t.x + a.t.y, buf[2], sum);
  if constexpr (TOP) top_threshold(k, top);
  __syncthreads();
  float s = 0.f, tt = 0.f;
  if (tid < 32) {   // what the threads that write results need
    s = reduce_block(buf[1], sum);
    if (ENT) tt = reduce_block(buf[2], sum);
  }
  if constexpr (TOP) top_of_part(p, my_max, k, top);
  if constexpr (SPLIT) {
    cluster_wait();   // the first block runs
    Joined* to = cluster.map_shared_rank(&joined, 0);
    if (tid == 0) {
      to->m[q] = m;
      to->s[q] = s;
      to->t[q] = tt;
    }
    if constexpr (TOP) {
      if (tid < k) to->best[q * k + tid] = top.best[tid];
    }
    cluster_arrive();
    if (q != 0) return;
    cluster_wait();
    // the parts' sums, each relative to its own maximum, relative to the row's
    m = joined.m[0];
    for (unsigned b = 1; b < R; ++b) m = fmaxf(m, joined.m[b]);
    wide = is_wide(m, c);
    ref = reference(m, c);
    s = tt = 0.f;
    for (unsigned b = 0; b < R; ++b) {
      const float mb = joined.m[b], rb = reference(mb, c);
      const bool wb = is_wide(mb, c);
      // what a part's exponents lack of the row's: from the difference of the maxima
      // where either is wide, each with what its reference lacks of it
      const float of_part = wb ? 0.f : fmaf(mb, c, -rb), of_row = wide ? 0.f : fmaf(m, c, -ref);
      float d = wide || wb ? (mb - m) * c - of_part + of_row : rb - ref;
      d = mb == -INFINITY ? 0.f : fmaxf(d, kLowZ);
      const float f = ex2_approx(d);
      s += f * joined.s[b];
      tt += f * fmaf(joined.s[b], d, joined.t[b]);
    }
    if constexpr (TOP) {
      if (tid < k) top.best[tid] = 0;
      __syncthreads();
      rank_keys(joined.best, (int)R * k, top.best, k);
      __syncthreads();
    }
  }
  if (m == INFINITY) s = NAN;
  const bool empty = m == -INFINITY && s == 0.f;
  const float l2 = log2f(s);
  auto value = [&](float x) {
    if (empty) return -INFINITY;
    const float z = fmaf(x, c, -ref), d = x - m;
    if (!wide && !(z < -1e30f)) return kLn2 * (z - l2);
    // far below the maximum, z may overflow where the difference does not, and the
    // difference where its quotient does not
    return (d == -INFINITY && x != -INFINITY ? x * inv_t - m * inv_t : d * inv_t) - kLn2 * l2;
  };
  if (tid == 0) {
    (void)MSB_OK(in, kSiteLogprobToken, t, V);
    logp[r] = in ? value(xt) : NAN;
    if (ENT) {
      const float H = kLn2 * (l2 - tt / s);
      entropy[r] = empty || H < 0.f ? 0.f : H;
    }
    stats[r * 3 + 0] = m;
    stats[r * 3 + 1] = s;
    stats[r * 3 + 2] = tt;
  }
  if constexpr (TOP) {
    if (tid < k) {
      const unsigned long long b = top.best[tid];   // 0: a row of NaN
      top_tok[r * k + tid] = b == 0 ? 0 : key_index(b);
      top_logp[r * k + tid] = b == 0 ? NAN : value(value_of((unsigned)(b >> 32)));
    }
  }
}

// Blocks of a row (splits of them) write dx over its vectors.  p_i = 2^z_i / s,
// so with A = -G - gH H and B = -gH,
//   dx_i = p_i (A + B log p_i) / T = 2^z_i (a + b z_i)
// for b = B ln 2 / (s T) and a = (A - B ln 2 log2 s) / (s T); the entries of
// the token and the alternatives are written again afterwards.  Rows go from
// the last to the first: the end of the logits is what the forward left in L2.
// Bound by DRAM: 8192 x 50257 fp16 241 us, 2048 x 128256 bf16 162 (6.5 TB/s).
template <typename T, bool ENT>
__global__ void __launch_bounds__(kThreads)
logprob_bwd_kernel(const T* __restrict__ logits, long long ld, const long long* __restrict__ tok,
                   long long M, int V, float c, float inv_t, long long ignore_index, int k,
                   const long long* __restrict__ top_tok, const float* __restrict__ stats,
                   const float* __restrict__ g_logp, const float* __restrict__ g_ent,
                   const float* __restrict__ g_top, T* __restrict__ dx, long long ld_dx,
                   unsigned splits) {
  ::msb::pdl_begin();
  constexpr int N = Vec<T>::N;
  __shared__ long long at[kMaxK + 1];
  __shared__ float gr[kMaxK + 1];
  const long long r = M - 1 - blockIdx.x / splits;
  const T* row = logits + r * ld;
  T* drow = dx + r * ld_dx;
  const int tid = threadIdx.x;
  const Part<T> p(row, V, blockIdx.x % splits, splits);
  const int lo = p.first ? 0 : p.at(p.v0), hi = p.last ? V : p.at(p.v1);
  // vectors where the two rows are aligned alike
  const bool vec = ((reinterpret_cast<uintptr_t>(row) ^ reinterpret_cast<uintptr_t>(drow)) & 15) == 0;
  uint4* dmid = reinterpret_cast<uint4*>(drow + p.head);
  const long long t = tok[r];
  const bool ignored = t == ignore_index;
  const float m = ignored ? -INFINITY : stats[r * 3], s = ignored ? 0.f : stats[r * 3 + 1];
  if (m == -INFINITY && s == 0.f) {
    const T zero = from_f32<T>(0.f);
    if (vec) {
      for (int v = p.v0 + tid; v < p.v1; v += kThreads) dmid[v] = make_uint4(0, 0, 0, 0);
      if (tid < p.loose()) drow[p.loose_at(tid)] = zero;
    } else {
      for (int i = lo + tid; i < hi; i += kThreads) drow[i] = zero;
    }
    return;
  }
  if (tid == 0) {
    const bool in = t >= 0 && t < V && g_logp != nullptr;
    at[0] = in ? t : -1;
    gr[0] = in ? g_logp[r] : 0.f;
  } else if (tid <= k) {
    at[tid] = top_tok[r * k + tid - 1];
    gr[tid] = g_top[r * k + tid - 1];
  }
  __syncthreads();
  float G = 0.f;
  for (int j = 0; j <= k; ++j) G += gr[j];
  const float l2 = log2f(s), w = inv_t / s;
  float a = -G * w, b = 0.f;
  if (ENT) {
    const float gh = g_ent[r], H = kLn2 * (l2 - stats[r * 3 + 2] / s);
    b = -gh * kLn2 * w;
    a = (-G - gh * H) * w - b * l2;
  }
  const bool wide = is_wide(m, c);
  const float ref = reference(m, c);
  auto of_z = [&](float z) {
    if (ENT) z = max_nan(z, kLowZ);
    return ex2_approx(z) * (ENT ? fmaf(b, z, a) : a);
  };
  auto value = [&](float x) { return of_z(wide ? (x - m) * c : fmaf(x, c, -ref)); };
  if (vec && !wide) {
    constexpr int U = 4;
    for (int v = p.v0 + tid; v < p.v1; v += U * kThreads) {
      Vec<T> x[U];
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (v + u * kThreads < p.v1) x[u].r = p.mid[v + u * kThreads];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        float f[N];
        x[u].unpack(f);
#pragma unroll
        for (int j = 0; j < N; ++j) f[j] = of_z(fmaf(f[j], c, -ref));
        uint4 o;
        if constexpr (N == 8) {
          o = pack_u4<T>(f);
        } else {
          o = make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]),
                         __float_as_uint(f[3]));
        }
        if (v + u * kThreads < p.v1) dmid[v + u * kThreads] = o;
      }
    }
    if (tid < p.loose()) {
      const int i = p.loose_at(tid);
      drow[i] = from_f32<T>(value(to_f32(row[i])));
    }
  } else {
    for (int i = lo + tid; i < hi; i += kThreads) drow[i] = from_f32<T>(value(to_f32(row[i])));
  }
  __syncthreads();
  if (tid <= k && at[tid] >= lo && at[tid] < hi) {
    float g = 0.f;
    bool first = true;
    for (int j = 0; j <= k; ++j) {
      if (at[j] != at[tid]) continue;
      first = first && j >= tid;
      g += gr[j];
    }
    if (first) {
      const int i = (int)at[tid];
      drow[i] = from_f32<T>(value(to_f32(row[i])) + g * inv_t);
    }
  }
}

// Blocks a row: up to `a_sm` a SM in all where rows are few, as long as a block has
// two vectors a thread.  The forward's blocks wait for one another: as many as are
// resident together, no more (96 x 128256 bf16 with 20 alternatives, in a graph:
// 21 us with one, 15 with two or four, 23 with eight; 2048 rows with their entropy:
// 92 us with one, 119 with two).  The backward's are independent, and even out the
// last rows (2048 rows: 172 us with one, 162 with two).
unsigned blocks_a_row(long long M, int V, int per_vec, int a_sm) {
  unsigned R = 1;
  while (R < kMaxCluster && M * 2 * R <= a_sm * kNumSMs && V / (int)(2 * R) >= per_vec * kThreads)
    R *= 2;
  return R;
}

}  // namespace

void logprob_fwd(const void* logits, long long ld, const long long* tok, long long M, int V,
                 float temperature, long long ignore_index, int k, float* logp, float* entropy,
                 float* top_logp, long long* top_tok, float* stats, int dtype, cudaStream_t st) {
  if (M == 0) return;
  const float c = (float)(1.4426950408889634 / (double)temperature);
  const float inv_t = (float)(1.0 / (double)temperature);
  MSB_DISPATCH_FLOAT(dtype, T, {
    const unsigned R = blocks_a_row(M, V, Vec<T>::N, 3);
    auto go = [&](auto ent, auto top) {
      constexpr bool E = decltype(ent)::value, K = decltype(top)::value;
      auto run = [&](auto* kernel) {
        launch_cluster(R, kernel, (unsigned)M * R, kThreads, 0, st, (const T*)logits, ld, tok, V, c,
                       inv_t, ignore_index, k, logp, entropy, top_logp, top_tok, stats);
      };
      R > 1 ? run(logprob_fwd_kernel<T, E, K, true>) : run(logprob_fwd_kernel<T, E, K, false>);
    };
    if (entropy != nullptr) {
      k > 0 ? go(std::true_type{}, std::true_type{}) : go(std::true_type{}, std::false_type{});
    } else {
      k > 0 ? go(std::false_type{}, std::true_type{}) : go(std::false_type{}, std::false_type{});
    }
  });
  MSB_CHECK_LAUNCH("logprob_fwd");
}

void logprob_bwd(const void* logits, long long ld, const long long* tok, long long M, int V,
                 float temperature, long long ignore_index, int k, const long long* top_tok,
                 const float* stats, const float* g_logp, const float* g_ent, const float* g_top,
                 void* dx, long long ld_dx, int dtype, cudaStream_t st) {
  if (M == 0) return;
  const float c = (float)(1.4426950408889634 / (double)temperature);
  const float inv_t = (float)(1.0 / (double)temperature);
  MSB_DISPATCH_FLOAT(dtype, T, {
    const unsigned R = blocks_a_row(M, V, Vec<T>::N, 32);
    auto go = [&](auto* kernel) {
      launch(kernel, (unsigned)M * R, kThreads, 0, st, (const T*)logits, ld, tok, M, V, c, inv_t,
             ignore_index, k, top_tok, stats, g_logp, g_ent, g_top, (T*)dx, ld_dx, R);
    };
    g_ent != nullptr ? go(logprob_bwd_kernel<T, true>) : go(logprob_bwd_kernel<T, false>);
  });
  MSB_CHECK_LAUNCH("logprob_bwd");
}

}  // namespace msb
