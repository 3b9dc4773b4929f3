// Log probabilities of given tokens, with the entropy of every position and
// its most probable alternatives, over model-dtype logits; and their gradient.
//
// Row x[0..V), temperature T, c = log2(e) / T, m = max(x), z_i = (x_i - m) c:
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
#include "common.cuh"
#include "vec.cuh"

namespace msb {

MSB_BOUNDS_TU(logprob)

namespace {

constexpr int kThreads = 512;

// (value, index) as one number: larger value first, then the lower index.
// NaN has no place in the order (0).
__device__ __forceinline__ unsigned long long key_of(float v, int i) {
  if (v != v) return 0ull;
  const int b = __float_as_int(v + 0.f);  // -0 counts as 0
  const unsigned u = b < 0 ? ~(unsigned)b : (unsigned)b | 0x80000000u;
  return ((unsigned long long)u << 32) | (0xffffffffu - (unsigned)i);
}
__device__ __forceinline__ int key_index(unsigned long long k) {
  return (int)(0xffffffffu - (unsigned)k);
}

__device__ __forceinline__ unsigned long long warp_max(unsigned long long v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const unsigned long long w = __shfl_xor_sync(0xffffffffu, v, o);
    v = w > v ? w : v;
  }
  return v;
}

// running maximum m of the logits, and the sums s, t relative to it.  The
// difference of two logits is taken before it is scaled: the lowest value of
// fp32 or bf16, a common mask, times c overflows.
struct Sums {
  float m, s, t;
};
// weight of a sum whose maximum lies d below the new one
__device__ __forceinline__ void scale_down(float& s, float& t, float d) {
  const float f = ex2_approx(d);
  t = f == 0.f ? 0.f : f * (t + s * d);
  s *= f;
}
__device__ __forceinline__ void add(Sums& a, float x, float c) {
  if (x > a.m) {
    if (a.m != -INFINITY) scale_down(a.s, a.t, (a.m - x) * c);
    a.s += 1.f;
    a.m = x;
  } else if (x != -INFINITY) {  // NaN as well
    const float z = (x - a.m) * c, e = ex2_approx(z);
    a.s += e;
    a.t += e == 0.f ? 0.f : e * z;
  }
}
__device__ __forceinline__ Sums merge(Sums a, Sums b, float c) {
  const float m = fmaxf(a.m, b.m);
  if (a.m != -INFINITY) scale_down(a.s, a.t, (a.m - m) * c);
  if (b.m != -INFINITY) scale_down(b.s, b.t, (b.m - m) * c);
  return {m, a.s + b.s, a.t + b.t};
}
__device__ __forceinline__ Sums warp_merge(Sums v, float c) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const Sums w = {__shfl_xor_sync(0xffffffffu, v.m, o), __shfl_xor_sync(0xffffffffu, v.s, o),
                    __shfl_xor_sync(0xffffffffu, v.t, o)};
    v = merge(v, w, c);
  }
  return v;
}

// One block a row: one pass for the sums, k more for the k alternatives.
template <typename T>
__global__ void __launch_bounds__(kThreads)
logprob_fwd_kernel(const T* __restrict__ logits, long long ld, const long long* __restrict__ tok,
                   int V, float c, float inv_t, long long ignore_index, int k,
                   float* __restrict__ logp,
                   float* __restrict__ entropy, float* __restrict__ top_logp,
                   long long* __restrict__ top_tok, float* __restrict__ stats) {
  ::msb::pdl_begin();
  __shared__ Sums part[32];
  __shared__ unsigned long long best[32];
  const long long r = blockIdx.x;
  const T* row = logits + r * ld;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, nw = blockDim.x >> 5;
  const long long t = tok[r];
  if (t == ignore_index) {
    if (threadIdx.x == 0) {
      logp[r] = 0.f;
      if (entropy != nullptr) entropy[r] = 0.f;
    }
    for (int j = threadIdx.x; j < k; j += blockDim.x) {
      top_logp[r * k + j] = 0.f;
      top_tok[r * k + j] = -1;
    }
    return;
  }
  Sums a = {-INFINITY, 0.f, 0.f};
  for (int i = threadIdx.x; i < V; i += blockDim.x) add(a, to_f32(row[i]), c);
  a = warp_merge(a, c);
  if (lane == 0) part[warp] = a;
  __syncthreads();
  a = part[0];
  for (int w = 1; w < nw; ++w) a = merge(a, part[w], c);
  if (a.m == INFINITY) a.s = NAN;
  const bool empty = a.m == -INFINITY && a.s == 0.f;
  const float l2 = log2f(a.s);
  const float H = kLn2 * (l2 - a.t / a.s);
  if (threadIdx.x == 0) {
    const bool in = MSB_OK(t >= 0 && t < V, kSiteLogprobToken, t, V);
    logp[r] = !in ? NAN : empty ? -INFINITY : (to_f32(row[t]) - a.m) * inv_t - kLn2 * l2;
    if (entropy != nullptr) entropy[r] = empty || H < 0.f ? 0.f : H;
    stats[r * 3 + 0] = a.m;
    stats[r * 3 + 1] = a.s;
    stats[r * 3 + 2] = a.t;
  }
  unsigned long long last = ~0ull;
  for (int j = 0; j < k; ++j) {
    unsigned long long b = 0;
    for (int i = threadIdx.x; i < V; i += blockDim.x) {
      const unsigned long long q = key_of(to_f32(row[i]), i);
      if (q < last && q > b) b = q;
    }
    b = warp_max(b);
    __syncthreads();
    if (lane == 0) best[warp] = b;
    __syncthreads();
    b = best[0];
    for (int w = 1; w < nw; ++w) b = best[w] > b ? best[w] : b;
    last = b;
    if (threadIdx.x == 0) {
      const int i = b == 0 ? 0 : key_index(b);
      top_tok[r * k + j] = i;
      top_logp[r * k + j] =
          empty ? -INFINITY : (to_f32(row[i]) - a.m) * inv_t - kLn2 * l2;
    }
  }
}

// One block a row.  p_i = 2^z_i / s, so with A = -G - gH H and B = -gH,
//   dx_i = p_i (A + B log p_i) / T = 2^z_i (a + b z_i)
// for b = B ln 2 / (s T) and a = (A - B ln 2 log2 s) / (s T); the entries of
// the token and the alternatives are written again afterwards.
template <typename T>
__global__ void __launch_bounds__(kThreads)
logprob_bwd_kernel(const T* __restrict__ logits, long long ld, const long long* __restrict__ tok,
                   int V, float c, float inv_t, long long ignore_index, int k,
                   const long long* __restrict__ top_tok, const float* __restrict__ stats,
                   const float* __restrict__ g_logp, const float* __restrict__ g_ent,
                   const float* __restrict__ g_top, T* __restrict__ dx, long long ld_dx) {
  ::msb::pdl_begin();
  __shared__ long long at[33];
  __shared__ float gr[33];
  const long long r = blockIdx.x;
  const T* row = logits + r * ld;
  T* drow = dx + r * ld_dx;
  const long long t = tok[r];
  const float m = stats[r * 3], s = stats[r * 3 + 1], tt = stats[r * 3 + 2];
  if (t == ignore_index || (m == -INFINITY && s == 0.f)) {
    for (int i = threadIdx.x; i < V; i += blockDim.x) drow[i] = from_f32<T>(0.f);
    return;
  }
  if (threadIdx.x == 0) {
    const bool in = t >= 0 && t < V && g_logp != nullptr;
    at[0] = in ? t : -1;
    gr[0] = in ? g_logp[r] : 0.f;
  } else if (threadIdx.x <= k) {
    at[threadIdx.x] = g_top != nullptr ? top_tok[r * k + threadIdx.x - 1] : -1;
    gr[threadIdx.x] = g_top != nullptr ? g_top[r * k + threadIdx.x - 1] : 0.f;
  }
  __syncthreads();
  float G = 0.f;
  for (int j = 0; j <= k; ++j) G += gr[j];
  const float gh = g_ent != nullptr ? g_ent[r] : 0.f;
  const float l2 = log2f(s), H = kLn2 * (l2 - tt / s), w = inv_t / s;
  const float b = -gh * kLn2 * w, a = (-G - gh * H) * w - b * l2;
  auto value = [&](int i) {
    const float z = fmaxf((to_f32(row[i]) - m) * c, -1e30f);
    return ex2_approx(z) * (a + b * z);
  };
  for (int i = threadIdx.x; i < V; i += blockDim.x) {
    const float v = to_f32(row[i]);
    drow[i] = from_f32<T>(v != v ? NAN : value(i));
  }
  __syncthreads();
  if (threadIdx.x <= k && at[threadIdx.x] >= 0) {
    float g = 0.f;
    bool first = true;
    for (int j = 0; j <= k; ++j) {
      if (at[j] != at[threadIdx.x]) continue;
      first = first && j >= (int)threadIdx.x;
      g += gr[j];
    }
    if (first) {
      const int i = (int)at[threadIdx.x];
      drow[i] = from_f32<T>(value(i) + g * inv_t);
    }
  }
}

}  // namespace

void logprob_fwd(const void* logits, long long ld, const long long* tok, long long M, int V,
                 float temperature, long long ignore_index, int k, float* logp, float* entropy,
                 float* top_logp, long long* top_tok, float* stats, int dtype, cudaStream_t st) {
  if (M == 0) return;
  const float c = (float)(1.4426950408889634 / (double)temperature);
  MSB_DISPATCH_FLOAT(dtype, T, {
    launch(logprob_fwd_kernel<T>, (unsigned)M, kThreads, 0, st, (const T*)logits, ld, tok, V, c,
           (float)(1.0 / temperature), ignore_index, k, logp, entropy, top_logp, top_tok, stats);
  });
  MSB_CHECK_LAUNCH("logprob_fwd");
}

void logprob_bwd(const void* logits, long long ld, const long long* tok, long long M, int V,
                 float temperature, long long ignore_index, int k, const long long* top_tok,
                 const float* stats, const float* g_logp, const float* g_ent, const float* g_top,
                 void* dx, long long ld_dx, int dtype, cudaStream_t st) {
  if (M == 0) return;
  const double c = 1.4426950408889634 / (double)temperature;
  MSB_DISPATCH_FLOAT(dtype, T, {
    launch(logprob_bwd_kernel<T>, (unsigned)M, kThreads, 0, st, (const T*)logits, ld, tok, V,
           (float)c, (float)(1.0 / temperature), ignore_index, k, top_tok, stats, g_logp, g_ent,
           g_top, (T*)dx, ld_dx);
  });
  MSB_CHECK_LAUNCH("logprob_bwd");
}

}  // namespace msb
