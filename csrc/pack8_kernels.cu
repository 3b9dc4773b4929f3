// Activations held in 8 bits between the forward and the backward pass.
//
// A row is cut into blocks of 32 values (the last one of a row may be short).
// A block is stored as a byte b, the exponent of its scale, and one signed
// byte q per value:
//
//   b = max(E(max |x|) - 6, 0)      E: the biased fp32 exponent field
//   q = clamp(rint(x * 2^(127 - b)), -127, 127)         x^ = q * 2^(b - 127)
//
// A power of two scales exactly, so rounding to q is the only rounding:
// |x^ - x| is at most half a step of 2^(b - 127), which is at most 2^-7 of the
// block's largest magnitude (a whole step where the largest rounds to 128).
// 127 steps stay below the next power of two, by enough to be finite in the
// type that the block came from.  A block that holds an infinity or a NaN gets b = 255 and comes back
// as NaN, so that an overflow check on the gradients sees it.
//
// Layout: codes [rows, 32 * nb], scales [rows, nb], nb = ceil(D / 32); a short
// last block is filled up with zero codes, so every block of codes is
// 32-byte aligned whatever D is.
#include "common.cuh"
#include "vec.cuh"

namespace msb {
namespace {

constexpr int kBlk = 32;      // values per scale
constexpr float kMagic = 12582912.f;  // 1.5 * 2^23: adding it leaves rint(x) in the low mantissa bits

__device__ __forceinline__ unsigned abs_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }

// scale byte of a block whose largest |x| has these bits
__device__ __forceinline__ unsigned scale_byte(unsigned amax) {
  const unsigned e = amax >> 23;
  return e == 255u ? 255u : (e > 6u ? e - 6u : 0u);
}
// 2^(127 - b); b <= 248 or 255 (whose codes are never read as numbers)
__device__ __forceinline__ float code_mul(unsigned b) {
  return __uint_as_float(b == 255u ? 0u : (254u - b) << 23);
}
// 2^(b - 127), NaN for 255
__device__ __forceinline__ float code_scale(unsigned b) {
  return b == 255u ? __uint_as_float(0x7fc00000u)
                   : __uint_as_float(b == 0u ? 0x00400000u : b << 23);
}
// q in the low byte of the result
__device__ __forceinline__ unsigned code_of(float x, float mul) {
  const float t = fmaf(x, mul, kMagic);
  return __float_as_uint(fminf(fmaxf(t, kMagic - 127.f), kMagic + 127.f));
}
__device__ __forceinline__ unsigned bytes4(unsigned a, unsigned b, unsigned c, unsigned d) {
  return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
}
// byte j of w as a number: 2^23 + (q + 128), minus 2^23 + 128
__device__ __forceinline__ float code_value(unsigned w, int j) {
  const unsigned bits = __byte_perm(w ^ 0x80808080u, 0x4b000000u, 0x7440 + j);
  return __uint_as_float(bits) - 8388736.f;
}

__device__ __forceinline__ uint2 codes8(const float (&f)[8], float mul) {
  unsigned q[8];
#pragma unroll
  for (int k = 0; k < 8; ++k) q[k] = code_of(f[k], mul);
  return make_uint2(bytes4(q[0], q[1], q[2], q[3]), bytes4(q[4], q[5], q[6], q[7]));
}
__device__ __forceinline__ void values8(uint2 w, float scale, float (&f)[8]) {
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    f[k] = code_value(w.x, k) * scale;
    f[4 + k] = code_value(w.y, k) * scale;
  }
}
__device__ __forceinline__ unsigned amax8(const float (&f)[8]) {
  unsigned m = 0;
#pragma unroll
  for (int k = 0; k < 8; ++k) m = max(m, abs_bits(f[k]));
  // the block's four lanes
  m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));
  return max(m, __shfl_xor_sync(0xffffffffu, m, 2));
}

// The vector kernels: widths that are a multiple of 8 and 16-byte aligned rows,
// four lanes a block, eight values a lane.  A thread has two vectors in flight,
// a grid's width apart.  The number of vectors of a launch fits 31 bits.
constexpr int kThreads = 256;
constexpr int kFlight = 2;

template <typename T>
__global__ void __launch_bounds__(kThreads)
pack8_vec_kernel(const T* __restrict__ x, long long ld, unsigned total, int D, FastDiv nv,
                 uint2* __restrict__ codes, unsigned char* __restrict__ scales) {
  ::msb::pdl_begin();
  const unsigned lane = threadIdx.x & 31, step = gridDim.x * kThreads;
  for (unsigned i0 = blockIdx.x * kThreads + threadIdx.x; i0 - lane < total; i0 += kFlight * step) {
    float f[kFlight][8];
#pragma unroll
    for (int u = 0; u < kFlight; ++u) {
      const unsigned i = i0 + u * step, row = nv.div(i), c = (i - row * nv.d) * 8;
#pragma unroll
      for (int k = 0; k < 8; ++k) f[u][k] = 0.f;
      if (i < total && c < D) load8(x + row * ld + c, f[u]);
    }
#pragma unroll
    for (int u = 0; u < kFlight; ++u) {
      const unsigned i = i0 + u * step;
      const unsigned b = scale_byte(amax8(f[u]));
      if (i < total) {
        codes[i] = codes8(f[u], code_mul(b));
        if ((lane & 3) == 0) scales[i >> 2] = (unsigned char)b;
      }
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(kThreads)
unpack8_vec_kernel(const uint2* __restrict__ codes, const unsigned char* __restrict__ scales,
                   T* __restrict__ x, unsigned total, int D, FastDiv nv) {
  ::msb::pdl_begin();
  const unsigned step = gridDim.x * kThreads;
  for (unsigned i0 = blockIdx.x * kThreads + threadIdx.x; i0 < total; i0 += kFlight * step) {
    uint2 w[kFlight];
    unsigned b[kFlight];
#pragma unroll
    for (int u = 0; u < kFlight; ++u) {
      const unsigned i = i0 + u * step;
      if (i >= total) continue;
      w[u] = codes[i];
      b[u] = scales[i >> 2];
    }
#pragma unroll
    for (int u = 0; u < kFlight; ++u) {
      const unsigned i = i0 + u * step, row = nv.div(i), c = (i - row * nv.d) * 8;
      if (i >= total || c >= D) continue;
      float f[8];
      values8(w[u], code_scale(b[u]), f);
      store8(x + (long long)row * D + c, f);
    }
  }
}

// Any width, stride and alignment: a warp a block, a value a lane.
template <typename T>
__global__ void __launch_bounds__(256)
pack8_any_kernel(const T* __restrict__ x, long long ld, long long blocks, int D, int nb,
                 signed char* __restrict__ codes, unsigned char* __restrict__ scales) {
  ::msb::pdl_begin();
  const int lane = threadIdx.x & 31;
  const long long step = (long long)gridDim.x * (blockDim.x >> 5);
  for (long long j = (long long)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5); j < blocks;
       j += step) {
    const long long row = j / nb;
    const int c = (int)(j - row * nb) * kBlk + lane;
    const float f = c < D ? to_f32(x[row * ld + c]) : 0.f;
    const unsigned b = scale_byte(__reduce_max_sync(0xffffffffu, abs_bits(f)));
    codes[j * kBlk + lane] = (signed char)(code_of(f, code_mul(b)) & 255u);
    if (lane == 0) scales[j] = (unsigned char)b;
  }
}

template <typename T>
__global__ void __launch_bounds__(256)
unpack8_any_kernel(const signed char* __restrict__ codes, const unsigned char* __restrict__ scales,
                   T* __restrict__ x, long long blocks, int D, int nb) {
  ::msb::pdl_begin();
  const int lane = threadIdx.x & 31;
  const long long step = (long long)gridDim.x * (blockDim.x >> 5);
  for (long long j = (long long)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5); j < blocks;
       j += step) {
    const long long row = j / nb;
    const int c = (int)(j - row * nb) * kBlk + lane;
    if (c < D) x[row * D + c] = from_f32<T>((float)codes[j * kBlk + lane] * code_scale(scales[j]));
  }
}

// quotients by __fdividef: 2 units in the last place, and 0 where 1 + e^-g
// passes 2^126, as the rounded quotient nearly is
__device__ __forceinline__ float silu_f(float g) { return __fdividef(g, 1.f + __expf(-g)); }
// h = silu(g) u:  dg = dh u s (1 + g (1 - s)),  du = dh g s,  s = sigmoid(g)
__device__ __forceinline__ void swiglu_grad(float dh, float g, float u, float& dg, float& du) {
  const float s = __fdividef(1.f, 1.f + __expf(-g));
  dg = dh * u * s * (1.f + g * (1.f - s));
  du = dh * g * s;
}

// gu rows are [gate (F) | up (F)]; the two halves are packed as rows 2r and
// 2r + 1 of width F, so each has blocks of its own.  Without codes (nullptr)
// only h is written.
template <typename T>
__global__ void __launch_bounds__(kThreads)
swiglu8_fwd_vec_kernel(const T* __restrict__ gu, T* __restrict__ h, uint2* __restrict__ codes,
                       unsigned char* __restrict__ scales, unsigned total, int F, FastDiv nv) {
  ::msb::pdl_begin();
  const unsigned lane = threadIdx.x & 31, step = gridDim.x * kThreads;
  for (unsigned i0 = blockIdx.x * kThreads + threadIdx.x; i0 - lane < total; i0 += kFlight * step) {
    float g[kFlight][8], u[kFlight][8];
#pragma unroll
    for (int j = 0; j < kFlight; ++j) {
      const unsigned i = i0 + j * step, row = nv.div(i), c = (i - row * nv.d) * 8;
#pragma unroll
      for (int k = 0; k < 8; ++k) g[j][k] = u[j][k] = 0.f;
      if (i < total && c < F) {
        load8(gu + (long long)row * 2 * F + c, g[j]);
        load8(gu + (long long)row * 2 * F + F + c, u[j]);
      }
    }
#pragma unroll
    for (int j = 0; j < kFlight; ++j) {
      const unsigned i = i0 + j * step, row = nv.div(i), v = i - row * nv.d, c = v * 8;
      const unsigned bg = scale_byte(amax8(g[j])), bu = scale_byte(amax8(u[j]));
      if (codes != nullptr && i < total) {
        const long long at = (long long)row * 2 * nv.d + v;
        codes[at] = codes8(g[j], code_mul(bg));
        codes[at + nv.d] = codes8(u[j], code_mul(bu));
        if ((lane & 3) == 0) {
          scales[at >> 2] = (unsigned char)bg;
          scales[(at + nv.d) >> 2] = (unsigned char)bu;
        }
      }
      if (i < total && c < F) {
#pragma unroll
        for (int k = 0; k < 8; ++k) g[j][k] = silu_f(g[j][k]) * u[j][k];
        store8(h + (long long)row * F + c, g[j]);
      }
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(kThreads)
swiglu8_bwd_vec_kernel(const T* __restrict__ dh, const uint2* __restrict__ codes,
                       const unsigned char* __restrict__ scales, T* __restrict__ dgu,
                       unsigned total, int F, FastDiv nv) {
  ::msb::pdl_begin();
  const unsigned step = gridDim.x * kThreads;
  for (unsigned i0 = blockIdx.x * kThreads + threadIdx.x; i0 < total; i0 += kFlight * step) {
    float d[kFlight][8];
    uint2 wg[kFlight], wu[kFlight];
    unsigned bg[kFlight], bu[kFlight];
#pragma unroll
    for (int j = 0; j < kFlight; ++j) {
      const unsigned i = i0 + j * step, row = nv.div(i), v = i - row * nv.d, c = v * 8;
      if (i >= total || c >= F) continue;
      const long long at = (long long)row * 2 * nv.d + v;
      wg[j] = codes[at];
      wu[j] = codes[at + nv.d];
      bg[j] = scales[at >> 2];
      bu[j] = scales[(at + nv.d) >> 2];
      load8(dh + (long long)row * F + c, d[j]);
    }
#pragma unroll
    for (int j = 0; j < kFlight; ++j) {
      const unsigned i = i0 + j * step, row = nv.div(i), c = (i - row * nv.d) * 8;
      if (i >= total || c >= F) continue;
      float g[8], u[8];
      values8(wg[j], code_scale(bg[j]), g);
      values8(wu[j], code_scale(bu[j]), u);
#pragma unroll
      for (int k = 0; k < 8; ++k) swiglu_grad(d[j][k], g[k], u[k], g[k], u[k]);
      store8(dgu + (long long)row * 2 * F + c, g);
      store8(dgu + (long long)row * 2 * F + F + c, u);
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(256)
swiglu8_fwd_any_kernel(const T* __restrict__ gu, T* __restrict__ h,
                       signed char* __restrict__ codes, unsigned char* __restrict__ scales,
                       long long blocks, int F, int nb) {
  ::msb::pdl_begin();
  const int lane = threadIdx.x & 31;
  const long long step = (long long)gridDim.x * (blockDim.x >> 5);
  for (long long j = (long long)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5); j < blocks;
       j += step) {
    const long long row = j / nb;
    const int k = (int)(j - row * nb), c = k * kBlk + lane;
    const float g = c < F ? to_f32(gu[row * 2 * F + c]) : 0.f;
    const float u = c < F ? to_f32(gu[row * 2 * F + F + c]) : 0.f;
    const unsigned bg = scale_byte(__reduce_max_sync(0xffffffffu, abs_bits(g)));
    const unsigned bu = scale_byte(__reduce_max_sync(0xffffffffu, abs_bits(u)));
    const long long at = row * 2 * nb + k;
    if (codes != nullptr) {
      codes[at * kBlk + lane] = (signed char)(code_of(g, code_mul(bg)) & 255u);
      codes[(at + nb) * kBlk + lane] = (signed char)(code_of(u, code_mul(bu)) & 255u);
      if (lane == 0) {
        scales[at] = (unsigned char)bg;
        scales[at + nb] = (unsigned char)bu;
      }
    }
    if (c < F) h[row * F + c] = from_f32<T>(silu_f(g) * u);
  }
}

template <typename T>
__global__ void __launch_bounds__(256)
swiglu8_bwd_any_kernel(const T* __restrict__ dh, const signed char* __restrict__ codes,
                       const unsigned char* __restrict__ scales, T* __restrict__ dgu,
                       long long blocks, int F, int nb) {
  ::msb::pdl_begin();
  const int lane = threadIdx.x & 31;
  const long long step = (long long)gridDim.x * (blockDim.x >> 5);
  for (long long j = (long long)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5); j < blocks;
       j += step) {
    const long long row = j / nb;
    const int k = (int)(j - row * nb), c = k * kBlk + lane;
    if (c >= F) continue;
    const long long at = row * 2 * nb + k;
    const float g = (float)codes[at * kBlk + lane] * code_scale(scales[at]);
    const float u = (float)codes[(at + nb) * kBlk + lane] * code_scale(scales[at + nb]);
    float dg, du;
    swiglu_grad(to_f32(dh[row * F + c]), g, u, dg, du);
    dgu[row * 2 * F + c] = from_f32<T>(dg);
    dgu[row * 2 * F + F + c] = from_f32<T>(du);
  }
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// a grid of 256-thread blocks that fills the GPU, eight a SM, and loops
int loop_grid(long long threads) { return grid_for(threads, kThreads, kNumSMs * 8); }

// f(first row, rows) over parts of at most 2^30 vectors, nv a row
template <typename F>
void in_parts(long long rows, int nv, F&& f) {
  const long long most = (1LL << 30) / nv > 0 ? (1LL << 30) / nv : 1;
  for (long long r = 0; r < rows; r += most) f(r, rows - r < most ? rows - r : most);
}

}  // namespace

void pack8(const void* x, long long ld, signed char* codes, unsigned char* scales, long long rows,
           int D, int dtype, cudaStream_t st) {
  const int nb = (D + kBlk - 1) / kBlk;
  MSB_DISPATCH_FLOAT(dtype, T, {
    const T* in = (const T*)x;
    if (D % 8 == 0 && aligned16(x) && (ld * sizeof(T)) % 16 == 0) {
      in_parts(rows, nb * 4, [&](long long r, long long n) {
        launch(pack8_vec_kernel<T>, loop_grid(n * nb * 4 / kFlight), kThreads, 0, st, in + r * ld,
               ld, (unsigned)(n * nb * 4), D, FastDiv(nb * 4), (uint2*)(codes + r * nb * kBlk),
               scales + r * nb);
      });
    } else if (rows > 0) {
      launch(pack8_any_kernel<T>, loop_grid(rows * nb * 32), kThreads, 0, st, in, ld, rows * nb, D,
             nb, codes, scales);
    }
  });
  MSB_CHECK_LAUNCH("pack8");
}

void unpack8(const signed char* codes, const unsigned char* scales, void* x, long long rows, int D,
             int dtype, cudaStream_t st) {
  const int nb = (D + kBlk - 1) / kBlk;
  MSB_DISPATCH_FLOAT(dtype, T, {
    if (D % 8 == 0) {
      in_parts(rows, nb * 4, [&](long long r, long long n) {
        launch(unpack8_vec_kernel<T>, loop_grid(n * nb * 4 / kFlight), kThreads, 0, st,
               (const uint2*)(codes + r * nb * kBlk), scales + r * nb, (T*)x + r * D,
               (unsigned)(n * nb * 4), D, FastDiv(nb * 4));
      });
    } else if (rows > 0) {
      launch(unpack8_any_kernel<T>, loop_grid(rows * nb * 32), kThreads, 0, st, codes, scales,
             (T*)x, rows * nb, D, nb);
    }
  });
  MSB_CHECK_LAUNCH("unpack8");
}

void swiglu8_fwd(const void* gu, void* h, signed char* codes, unsigned char* scales,
                 long long rows, int F, int dtype, cudaStream_t st) {
  const int nb = (F + kBlk - 1) / kBlk;
  MSB_DISPATCH_FLOAT(dtype, T, {
    if (F % 8 == 0 && aligned16(gu)) {
      in_parts(rows, nb * 4, [&](long long r, long long n) {
        launch(swiglu8_fwd_vec_kernel<T>, loop_grid(n * nb * 4 / kFlight), kThreads, 0, st,
               (const T*)gu + r * 2 * F, (T*)h + r * F,
               codes == nullptr ? nullptr : (uint2*)(codes + r * 2 * nb * kBlk),
               scales + r * 2 * nb, (unsigned)(n * nb * 4), F, FastDiv(nb * 4));
      });
    } else if (rows > 0) {
      launch(swiglu8_fwd_any_kernel<T>, loop_grid(rows * nb * 32), kThreads, 0, st, (const T*)gu,
             (T*)h, codes, scales, rows * nb, F, nb);
    }
  });
  MSB_CHECK_LAUNCH("swiglu8_fwd");
}

void swiglu8_bwd(const void* dh, const signed char* codes, const unsigned char* scales, void* dgu,
                 long long rows, int F, int dtype, cudaStream_t st) {
  const int nb = (F + kBlk - 1) / kBlk;
  MSB_DISPATCH_FLOAT(dtype, T, {
    if (F % 8 == 0 && aligned16(dh)) {
      in_parts(rows, nb * 4, [&](long long r, long long n) {
        launch(swiglu8_bwd_vec_kernel<T>, loop_grid(n * nb * 4 / kFlight), kThreads, 0, st,
               (const T*)dh + r * F, (const uint2*)(codes + r * 2 * nb * kBlk),
               scales + r * 2 * nb, (T*)dgu + r * 2 * F, (unsigned)(n * nb * 4), F,
               FastDiv(nb * 4));
      });
    } else if (rows > 0) {
      launch(swiglu8_bwd_any_kernel<T>, loop_grid(rows * nb * 32), kThreads, 0, st, (const T*)dh,
             codes, scales, (T*)dgu, rows * nb, F, nb);
    }
  });
  MSB_CHECK_LAUNCH("swiglu8_bwd");
}

}  // namespace msb
