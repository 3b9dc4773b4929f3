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
// q in the low byte of the result; CLAMP: x may round to 128 steps
template <bool CLAMP = true>
__device__ __forceinline__ unsigned code_of(float x, float mul) {
  float t = fmaf(x, mul, kMagic);
  if (CLAMP) t = fminf(fmaxf(t, kMagic - 127.f), kMagic + 127.f);
  return __float_as_uint(t);
}
__device__ __forceinline__ unsigned bytes4(unsigned a, unsigned b, unsigned c, unsigned d) {
  return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
}
// byte j of w as a number: 2^23 + (q + 128), minus 2^23 + 128
__device__ __forceinline__ float code_value(unsigned w, int j) {
  const unsigned bits = __byte_perm(w ^ 0x80808080u, 0x4b000000u, 0x7440 + j);
  return __uint_as_float(bits) - 8388736.f;
}

template <bool CLAMP>
__device__ __forceinline__ uint2 codes8(const float (&f)[8], float mul) {
  unsigned q[8];
#pragma unroll
  for (int k = 0; k < 8; ++k) q[k] = code_of<CLAMP>(f[k], mul);
  return make_uint2(bytes4(q[0], q[1], q[2], q[3]), bytes4(q[4], q[5], q[6], q[7]));
}
__device__ __forceinline__ void values8(uint2 w, float scale, float (&f)[8]) {
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    f[k] = code_value(w.x, k) * scale;
    f[4 + k] = code_value(w.y, k) * scale;
  }
}

// Eight values of a row: as loaded, as numbers, and the largest magnitude
// (NaN where one is), in 16 bits two at a time.
template <typename T>
struct Eight {
  uint4 r;
  __device__ __forceinline__ void load(const T* p) { r = *reinterpret_cast<const uint4*>(p); }
  __device__ __forceinline__ void zero() { r = make_uint4(0, 0, 0, 0); }
  __device__ __forceinline__ void numbers(float (&f)[8]) const { unpack_u4<T>(r, f); }
  __device__ __forceinline__ float amax() const {
    if constexpr (std::is_same<T, __half>::value) {
      const __half2* p = reinterpret_cast<const __half2*>(&r);
      const __half2 m = __hmax2_nan(__hmax2_nan(__habs2(p[0]), __habs2(p[1])),
                                    __hmax2_nan(__habs2(p[2]), __habs2(p[3])));
      return max_nan(__low2float(m), __high2float(m));
    } else {
      const __nv_bfloat162* p = reinterpret_cast<const __nv_bfloat162*>(&r);
      const __nv_bfloat162 m = __hmax2_nan(__hmax2_nan(__habs2(p[0]), __habs2(p[1])),
                                           __hmax2_nan(__habs2(p[2]), __habs2(p[3])));
      return max_nan(__low2float(m), __high2float(m));
    }
  }
};
template <>
struct Eight<float> {
  float4 a, b;
  __device__ __forceinline__ void load(const float* p) {
    a = reinterpret_cast<const float4*>(p)[0];
    b = reinterpret_cast<const float4*>(p)[1];
  }
  __device__ __forceinline__ void zero() { a = b = make_float4(0.f, 0.f, 0.f, 0.f); }
  __device__ __forceinline__ void numbers(float (&f)[8]) const {
    f[0] = a.x, f[1] = a.y, f[2] = a.z, f[3] = a.w, f[4] = b.x, f[5] = b.y, f[6] = b.z, f[7] = b.w;
  }
  __device__ __forceinline__ float amax() const {
    return max_nan(max_nan(max_nan(fabsf(a.x), fabsf(a.y)), max_nan(fabsf(a.z), fabsf(a.w))),
                   max_nan(max_nan(fabsf(b.x), fabsf(b.y)), max_nan(fabsf(b.z), fabsf(b.w))));
  }
};
template <typename T>
__device__ __forceinline__ void store_eight(T* p, const float (&f)[8]) {
  if constexpr (sizeof(T) == 2) {
    *reinterpret_cast<uint4*>(p) = pack_u4<T>(f);
  } else {
    reinterpret_cast<float4*>(p)[0] = make_float4(f[0], f[1], f[2], f[3]);
    reinterpret_cast<float4*>(p)[1] = make_float4(f[4], f[5], f[6], f[7]);
  }
}

// The scale of a block from its four lanes' magnitudes: its byte, the codes'
// multiplier, and whether a value may round to 128 steps.
struct Scale {
  unsigned byte;
  float mul;
  bool clamp;
  __device__ __forceinline__ explicit Scale(float m) {
    m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, 1));
    m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, 2));
    byte = scale_byte(abs_bits(m));
    mul = code_mul(byte);
    clamp = m * mul >= 127.5f;
  }
};

// The vector kernels: widths that are a multiple of 8 and 16-byte aligned rows,
// four lanes a block, eight values a lane.  A thread has two vectors in flight,
// a grid's width apart.  The number of vectors of a launch fits 31 bits.
// Bound by DRAM: swiglu8 at 4096 x 14336 bf16 moves its 473 MB in 77 us forward
// and 80 us backward, 6.1 and 5.9 TB/s.
constexpr int kThreads = 256;
constexpr int kFlight = 2;

template <typename T>
__global__ void __launch_bounds__(kThreads)
pack8_vec_kernel(const T* __restrict__ x, long long ld, unsigned total, int D, FastDiv nv,
                 uint2* __restrict__ codes, unsigned char* __restrict__ scales) {
  ::msb::pdl_begin();
  const unsigned lane = threadIdx.x & 31, step = gridDim.x * kThreads;
  for (unsigned i0 = blockIdx.x * kThreads + threadIdx.x; i0 - lane < total; i0 += kFlight * step) {
    Eight<T> v[kFlight];
#pragma unroll
    for (int u = 0; u < kFlight; ++u) {
      const unsigned i = i0 + u * step, row = nv.div(i), c = (i - row * nv.d) * 8;
      v[u].zero();
      if (i < total && c < D) v[u].load(x + row * ld + c);
    }
#pragma unroll
    for (int u = 0; u < kFlight; ++u) {
      const unsigned i = i0 + u * step;
      const Scale s(v[u].amax());
      float f[8];
      v[u].numbers(f);
      // the clamp is worth a branch: about one block in 200 needs it
      const uint2 w = __any_sync(0xffffffffu, s.clamp) ? codes8<true>(f, s.mul)
                                                       : codes8<false>(f, s.mul);
      if (i < total) {
        codes[i] = w;
        if ((lane & 3) == 0) scales[i >> 2] = (unsigned char)s.byte;
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
      store_eight(x + (long long)row * D + c, f);
    }
  }
}

// Any width, stride and alignment: eight lanes a block, four values a lane,
// loaded and stored one by one.  The price against the vector kernels, at
// 16384 x 2047 beside 2048: bf16 pack 33 us beside 20, unpack 41 / 19, swiglu8
// forward 69 / 50, backward 79 / 51; fp32 37 / 29, 39 / 42, 87 / 77, 90 / 80.
template <typename T>
struct Four {
  float f[4];
  __device__ __forceinline__ void load(const T* p, int left) {   // left: values of the row from p on
#pragma unroll
    for (int k = 0; k < 4; ++k) f[k] = k < left ? to_f32(p[k]) : 0.f;
  }
  __device__ __forceinline__ void store(T* p, int left) const {
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (k < left) p[k] = from_f32<T>(f[k]);
  }
  __device__ __forceinline__ float amax() const {
    const float m = max_nan(max_nan(fabsf(f[0]), fabsf(f[1])), max_nan(fabsf(f[2]), fabsf(f[3])));
    return max_nan(m, __shfl_xor_sync(0xffffffffu, m, 4));
  }
  __device__ __forceinline__ unsigned codes(float mul) const {
    return bytes4(code_of(f[0], mul), code_of(f[1], mul), code_of(f[2], mul), code_of(f[3], mul));
  }
  __device__ __forceinline__ void values(unsigned w, float scale) {
#pragma unroll
    for (int k = 0; k < 4; ++k) f[k] = code_value(w, k) * scale;
  }
};

template <typename T>
__global__ void __launch_bounds__(kThreads)
pack8_any_kernel(const T* __restrict__ x, long long ld, unsigned total, int D, FastDiv nq,
                 unsigned* __restrict__ codes, unsigned char* __restrict__ scales) {
  ::msb::pdl_begin();
  const unsigned lane = threadIdx.x & 31, step = gridDim.x * kThreads;
  for (unsigned i = blockIdx.x * kThreads + threadIdx.x; i - lane < total; i += step) {
    const unsigned row = nq.div(i);
    const int c = (int)(i - row * nq.d) * 4;
    Four<T> v;
    v.load(x + row * ld + c, i < total ? D - c : 0);
    const Scale s(v.amax());
    if (i < total) {
      codes[i] = v.codes(s.mul);
      if ((lane & 7) == 0) scales[i >> 3] = (unsigned char)s.byte;
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(kThreads)
unpack8_any_kernel(const unsigned* __restrict__ codes, const unsigned char* __restrict__ scales,
                   T* __restrict__ x, unsigned total, int D, FastDiv nq) {
  ::msb::pdl_begin();
  const unsigned step = gridDim.x * kThreads;
  for (unsigned i = blockIdx.x * kThreads + threadIdx.x; i < total; i += step) {
    const unsigned row = nq.div(i);
    const int c = (int)(i - row * nq.d) * 4;
    Four<T> v;
    v.values(codes[i], code_scale(scales[i >> 3]));
    v.store(x + (long long)row * D + c, D - c);
  }
}

// sigmoid(g); 0 where e^-g overflows.  In 16 bits by approximations whose error,
// some 2^-24 |g| of the value, is far below the result's half step of 2^-11 or
// 2^-8 of it (in quarters, as the reciprocal of a number from 2^126 on is flushed
// to 0, and bf16 has values that small); fp32 has no such room and takes the
// exponential and the quotient that SwiGLU without 8-bit saves does.
template <typename T>
__device__ __forceinline__ float sigmoid_of(float g) {
  return sizeof(T) == 4 ? 1.f / (1.f + expf(-g))
                        : 0.25f * rcp_approx(fmaf(0.25f, ex2_approx(g * -kLog2e), 0.25f));
}
template <typename T>
__device__ __forceinline__ float silu_of(float g) {
  return sizeof(T) == 4 ? g / (1.f + expf(-g)) : g * sigmoid_of<T>(g);
}
// h = silu(g) u:  dg = dh u s (1 + g (1 - s)),  du = dh g s,  s = sigmoid(g).
// The smallest factor is s; times dh alone it may be subnormal where the results
// are not.
template <typename T>
__device__ __forceinline__ void swiglu_grad(float dh, float g, float u, float& dg, float& du) {
  const float s = sigmoid_of<T>(g);
  dg = dh * u * (s * fmaf(g, 1.f - s, 1.f));
  du = dh * (g * s);
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
    Eight<T> vg[kFlight], vu[kFlight];
#pragma unroll
    for (int j = 0; j < kFlight; ++j) {
      const unsigned i = i0 + j * step, row = nv.div(i), c = (i - row * nv.d) * 8;
      vg[j].zero();
      vu[j].zero();
      if (i < total && c < F) {
        const T* p = gu + (long long)row * 2 * F + c;
        vg[j].load(p);
        vu[j].load(p + F);
      }
    }
#pragma unroll
    for (int j = 0; j < kFlight; ++j) {
      const unsigned i = i0 + j * step, row = nv.div(i), v = i - row * nv.d, c = v * 8;
      float g[8], u[8];
      vg[j].numbers(g);
      vu[j].numbers(u);
      if (codes != nullptr) {
        const Scale sg(vg[j].amax()), su(vu[j].amax());
        uint2 wg, wu;
        // the clamp is worth a branch: about one block in 200 needs it
        if (__any_sync(0xffffffffu, sg.clamp || su.clamp)) {
          wg = codes8<true>(g, sg.mul);
          wu = codes8<true>(u, su.mul);
        } else {
          wg = codes8<false>(g, sg.mul);
          wu = codes8<false>(u, su.mul);
        }
        if (i < total) {
          const long long at = (long long)row * 2 * nv.d + v;
          codes[at] = wg;
          codes[at + nv.d] = wu;
          if ((lane & 3) == 0) {
            scales[at >> 2] = (unsigned char)sg.byte;
            scales[(at + nv.d) >> 2] = (unsigned char)su.byte;
          }
        }
      }
      if (i < total && c < F) {
#pragma unroll
        for (int k = 0; k < 8; ++k) g[k] = silu_of<T>(g[k]) * u[k];
        store_eight(h + (long long)row * F + c, g);
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
    Eight<T> vd[kFlight];
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
      vd[j].load(dh + (long long)row * F + c);
    }
#pragma unroll
    for (int j = 0; j < kFlight; ++j) {
      const unsigned i = i0 + j * step, row = nv.div(i), c = (i - row * nv.d) * 8;
      if (i >= total || c >= F) continue;
      float d[8], g[8], u[8];
      vd[j].numbers(d);
      values8(wg[j], code_scale(bg[j]), g);
      values8(wu[j], code_scale(bu[j]), u);
#pragma unroll
      for (int k = 0; k < 8; ++k) swiglu_grad<T>(d[k], g[k], u[k], g[k], u[k]);
      T* p = dgu + (long long)row * 2 * F + c;
      store_eight(p, g);
      store_eight(p + F, u);
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(kThreads)
swiglu8_fwd_any_kernel(const T* __restrict__ gu, T* __restrict__ h, unsigned* __restrict__ codes,
                       unsigned char* __restrict__ scales, unsigned total, int F, FastDiv nq) {
  ::msb::pdl_begin();
  const unsigned lane = threadIdx.x & 31, step = gridDim.x * kThreads;
  for (unsigned i = blockIdx.x * kThreads + threadIdx.x; i - lane < total; i += step) {
    const unsigned row = nq.div(i), v = i - row * nq.d;
    const int c = (int)v * 4, left = i < total ? F - c : 0;
    const T* p = gu + (long long)row * 2 * F + c;
    Four<T> g, u;
    g.load(p, left);
    u.load(p + F, left);
    if (codes != nullptr) {
      const Scale sg(g.amax()), su(u.amax());
      if (i < total) {
        const long long at = (long long)row * 2 * nq.d + v;
        codes[at] = g.codes(sg.mul);
        codes[at + nq.d] = u.codes(su.mul);
        if ((lane & 7) == 0) {
          scales[at >> 3] = (unsigned char)sg.byte;
          scales[(at + nq.d) >> 3] = (unsigned char)su.byte;
        }
      }
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) g.f[k] = silu_of<T>(g.f[k]) * u.f[k];
    g.store(h + (long long)row * F + c, left);
  }
}

template <typename T>
__global__ void __launch_bounds__(kThreads)
swiglu8_bwd_any_kernel(const T* __restrict__ dh, const unsigned* __restrict__ codes,
                       const unsigned char* __restrict__ scales, T* __restrict__ dgu,
                       unsigned total, int F, FastDiv nq) {
  ::msb::pdl_begin();
  const unsigned step = gridDim.x * kThreads;
  for (unsigned i = blockIdx.x * kThreads + threadIdx.x; i < total; i += step) {
    const unsigned row = nq.div(i), v = i - row * nq.d;
    const int c = (int)v * 4, left = F - c;
    const long long at = (long long)row * 2 * nq.d + v;
    Four<T> d, g, u;
    d.load(dh + (long long)row * F + c, left);
    g.values(codes[at], code_scale(scales[at >> 3]));
    u.values(codes[at + nq.d], code_scale(scales[(at + nq.d) >> 3]));
#pragma unroll
    for (int k = 0; k < 4; ++k) swiglu_grad<T>(d.f[k], g.f[k], u.f[k], g.f[k], u.f[k]);
    T* p = dgu + (long long)row * 2 * F + c;
    g.store(p, left);
    u.store(p + F, left);
  }
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// Grids of 256-thread blocks that loop, at most 16 a SM: calls of swiglu8_fwd at
// 4096 x 14336 bf16 took 78 us each with 16, 80 with 8, 82 with the 4 that are
// resident at once, 99 with 5 (a short second wave), and swiglu8_bwd 82, 87
// without a loop.
int loop_grid(long long threads) { return grid_for(threads, kThreads, kNumSMs * 16); }

// f(first row, rows, threads' units of work) over parts of at most 2^30 units
template <typename F>
void in_parts(long long rows, int units_a_row, F&& f) {
  const long long fit = (1LL << 30) / units_a_row, most = fit > 0 ? fit : 1;
  for (long long r = 0; r < rows; r += most) {
    const long long n = rows - r < most ? rows - r : most;
    f(r, n * units_a_row);
  }
}

int blocks_of(int width) { return (width + kBlk - 1) / kBlk; }

}  // namespace

void pack8(const void* x, long long ld, signed char* codes, unsigned char* scales, long long rows,
           int D, int dtype, cudaStream_t st) {
  const int nb = blocks_of(D);
  MSB_DISPATCH_FLOAT(dtype, T, {
    const bool vec = D % 8 == 0 && aligned16(x) && (ld * sizeof(T)) % 16 == 0;
    const int per = nb * (vec ? 4 : 8);
    in_parts(rows, per, [&](long long r, long long n) {
      const T* in = (const T*)x + r * ld;
      signed char* cd = codes + r * nb * kBlk;
      if (vec) {
        launch(pack8_vec_kernel<T>, loop_grid(n / kFlight), kThreads, 0, st, in, ld, (unsigned)n,
               D, FastDiv(per), (uint2*)cd, scales + r * nb);
      } else {
        launch(pack8_any_kernel<T>, loop_grid(n), kThreads, 0, st, in, ld, (unsigned)n, D,
               FastDiv(per), (unsigned*)cd, scales + r * nb);
      }
    });
  });
  MSB_CHECK_LAUNCH("pack8");
}

void unpack8(const signed char* codes, const unsigned char* scales, void* x, long long rows, int D,
             int dtype, cudaStream_t st) {
  const int nb = blocks_of(D);
  MSB_DISPATCH_FLOAT(dtype, T, {
    const bool vec = D % 8 == 0;
    const int per = nb * (vec ? 4 : 8);
    in_parts(rows, per, [&](long long r, long long n) {
      const signed char* cd = codes + r * nb * kBlk;
      T* out = (T*)x + r * D;
      if (vec) {
        launch(unpack8_vec_kernel<T>, loop_grid(n / kFlight), kThreads, 0, st, (const uint2*)cd,
               scales + r * nb, out, (unsigned)n, D, FastDiv(per));
      } else {
        launch(unpack8_any_kernel<T>, loop_grid(n), kThreads, 0, st, (const unsigned*)cd,
               scales + r * nb, out, (unsigned)n, D, FastDiv(per));
      }
    });
  });
  MSB_CHECK_LAUNCH("unpack8");
}

void swiglu8_fwd(const void* gu, void* h, signed char* codes, unsigned char* scales,
                 long long rows, int F, int dtype, cudaStream_t st) {
  const int nb = blocks_of(F);
  MSB_DISPATCH_FLOAT(dtype, T, {
    const bool vec = F % 8 == 0 && aligned16(gu);
    const int per = nb * (vec ? 4 : 8);
    in_parts(rows, per, [&](long long r, long long n) {
      const T* in = (const T*)gu + r * 2 * F;
      T* out = (T*)h + r * F;
      signed char* cd = codes == nullptr ? nullptr : codes + r * 2 * nb * kBlk;
      unsigned char* sc = scales + r * 2 * nb;
      if (vec) {
        launch(swiglu8_fwd_vec_kernel<T>, loop_grid(n / kFlight), kThreads, 0, st, in, out,
               (uint2*)cd, sc, (unsigned)n, F, FastDiv(per));
      } else {
        launch(swiglu8_fwd_any_kernel<T>, loop_grid(n), kThreads, 0, st, in, out, (unsigned*)cd,
               sc, (unsigned)n, F, FastDiv(per));
      }
    });
  });
  MSB_CHECK_LAUNCH("swiglu8_fwd");
}

void swiglu8_bwd(const void* dh, const signed char* codes, const unsigned char* scales, void* dgu,
                 long long rows, int F, int dtype, cudaStream_t st) {
  const int nb = blocks_of(F);
  MSB_DISPATCH_FLOAT(dtype, T, {
    const bool vec = F % 8 == 0 && aligned16(dh);
    const int per = nb * (vec ? 4 : 8);
    in_parts(rows, per, [&](long long r, long long n) {
      const T* in = (const T*)dh + r * F;
      T* out = (T*)dgu + r * 2 * F;
      const signed char* cd = codes + r * 2 * nb * kBlk;
      const unsigned char* sc = scales + r * 2 * nb;
      if (vec) {
        launch(swiglu8_bwd_vec_kernel<T>, loop_grid(n / kFlight), kThreads, 0, st, in,
               (const uint2*)cd, sc, out, (unsigned)n, F, FastDiv(per));
      } else {
        launch(swiglu8_bwd_any_kernel<T>, loop_grid(n), kThreads, 0, st, in, (const unsigned*)cd,
               sc, out, (unsigned)n, F, FastDiv(per));
      }
    });
  });
  MSB_CHECK_LAUNCH("swiglu8_bwd");
}

}  // namespace msb
