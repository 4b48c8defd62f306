// Activations kept in 8 bits for the backward pass, and GELU on them.
//
// Along the last axis every 128 values share the least power of two 2^e,
// e >= -126, with max|x| <= 127 * 2^e, and keep x / 2^e rounded to the
// nearest integer (ties to even).  A power of two makes the scaling exact:
// the one rounding is the integer's, at most half a step of max|x| / 63.5,
// and the stored value is exact in bfloat16, so a matrix product can take it
// as it is.  A value that would round to 2^128 is held as 63 * 2^122.
// (8-bit floats would spend bits on range that a block of 128
// activations does not have: on normal data their error is 2 to 4 times
// larger.)  A block with an infinity or NaN reads back as NaN.
//
//   gelu(x)  = x * Phi(x)
//   gelu'(x) = Phi(x) + x * phi(x)
//
// Bound by memory in fp32 (9 bytes a value each way) and close to the vector
// units' rate in bf16 (5 bytes): Phi is built from one exp and a short
// polynomial (in fp32 a second one near 0) instead of the library's two-branch
// erf, which alone takes longer than the bf16 traffic.  16 threads own a block of 128, 8 values
// each; the maximum crosses lanes by four shuffles.  Measured: 409600 x 512
// bf16 forward 237 us, backward 236 us, 4.4 TB/s both; 32768 x 1024 packed in
// 20 to 25 us.  Rows that are not whole 16-byte accesses are read value by
// value: 409600 x 509 bf16 forward 600 us, backward 571.

#include "token_ops.h"
#include "token_device.h"

#include <algorithm>

namespace token_ops {
namespace {

constexpr int kThreads = 256;

// Phi(-a) = exp(-a^2/2) * t * Q(t), t = 1 / (1 + c a), a >= 0: least-maximum
// fits of 0.5 * erfcx(a / sqrt(2)) / t.  Relative error 1.1e-5 in 5 degrees
// (bf16 output, half a step is 3.9e-3), 4e-7 in 8 (fp32).
template <typename T> __device__ __forceinline__ float tail_q(float t);
template <> __device__ __forceinline__ float tail_q<bf16>(float t) {
  float q = -0.06677515059709549f;
  q = fmaf(q, t, 0.13958728313446045f);
  q = fmaf(q, t, 0.04961274564266205f);
  q = fmaf(q, t, 0.12305187433958054f);
  q = fmaf(q, t, 0.12682804465293884f);
  return fmaf(q, t, 0.12768971920013428f);
}
template <> __device__ __forceinline__ float tail_q<float>(float t) {
  float q = -0.030238229781389236f;
  q = fmaf(q, t, 0.13950829207897186f);
  q = fmaf(q, t, -0.22359946370124817f);
  q = fmaf(q, t, 0.10736914724111557f);
  q = fmaf(q, t, -0.00038640544516965747f);
  q = fmaf(q, t, 0.0960373803973198f);
  q = fmaf(q, t, 0.12400975078344345f);
  q = fmaf(q, t, 0.14368188381195068f);
  return fmaf(q, t, 0.1436176598072052f);
}
template <typename T> struct TailC;
template <> struct TailC<bf16> { static constexpr float c = 0.32f; };
template <> struct TailC<float> { static constexpr float c = 0.36f; };

// Phi(x) and exp(-x^2/2)
template <typename T>
__device__ __forceinline__ float normal_cdf(float x, float& e) {
  const float a = fabsf(x);
  const float t = __builtin_amdgcn_rcpf(fmaf(TailC<T>::c, a, 1.f));
  e = __builtin_amdgcn_exp2f(a * a * -0.72134752044448170f);  // -log2(e)/2
  const float tail = e * (t * tail_q<T>(t));
  const float far = x < 0.f ? tail : 1.f - tail;
  if constexpr (sizeof(T) == 4) {
    // Near 0 the quotient's and the exponential's errors would show: there
    // Phi = 1/2 + x S(x^2), the series of the density's integral, up to
    // x^15 (2e-9 left at 1).  Relative error of x * Phi for |x| < 1 in half
    // steps of fp32: 0.8 on average and 4 at most, where the quotient alone
    // has 1.9 and 7.
    const float s = a * a;
    float q = -4.122667363e-8f;
    q = fmaf(q, s, 6.659693668e-7f);
    q = fmaf(q, s, -9.444655916e-6f);
    q = fmaf(q, s, 1.1543469009e-4f);
    q = fmaf(q, s, -1.1873282492e-3f);
    q = fmaf(q, s, 9.973556735e-3f);
    q = fmaf(q, s, -6.649038196e-2f);
    q = fmaf(q, s, 0.3989422917f);
    return a < 1.f ? fmaf(x, q, 0.5f) : far;
  } else {
    return far;
  }
}

// Biased exponent of the block whose largest |x| has these bits; 255 where
// it is not finite.  127 = 1.984375 * 2^6.
__device__ __forceinline__ uint32_t block_exponent(uint32_t top) {
  if (top >= 0x7f800000u) return 255u;
  const int f = (int)(top >> 23) - 6 + ((top & 0x7fffffu) > 0x7e0000u ? 1 : 0);
  return (uint32_t)(f < 1 ? 1 : f);
}

__device__ __forceinline__ void pack8(const float (&v)[8], uint32_t& e,
                                      u32x2& q) {
  uint32_t top = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j)
    top = max(top, __float_as_uint(v[j]) & 0x7fffffffu);
#pragma unroll
  for (int o = 1; o < 16; o <<= 1)
    top = max(top, (uint32_t)__shfl_xor((int)top, o, 64));
  e = block_exponent(top);
  const float inv = e == 255u ? 0.f : __uint_as_float((254u - e) << 23);
  // under the largest exponent 64 units would be 2^128, beyond fp32
  const float most = e == 249u ? 63.f : 127.f;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    uint32_t w = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      // a block that is not finite stores zeros: 0 * inf reads back as NaN
      const float r = fminf(fmaxf(rintf(v[4 * h + j] * inv), -most), most);
      const int n = e == 255u ? 0 : (int)r;
      w |= (uint32_t)(n & 0xff) << (8 * j);
    }
    q[h] = w;
  }
}

struct Chunk {        // 8 values of one row, `sub` of 16 in a block of 128
  long long row, blk;
  int col, sub;
};
// Blocks a row are `nb`; the common widths need no division.
__device__ __forceinline__ Chunk chunk_at(long long c, long long nb) {
  Chunk r;
  r.blk = c >> 4;
  r.sub = (int)(c & 15);
  r.row = nb == 1 ? r.blk : r.blk / nb;
  r.col = (int)(r.blk - r.row * nb) * 128 + r.sub * 8;
  return r;
}

template <typename T, bool VEC>
__device__ __forceinline__ void load8(const T* p, int valid, float (&v)[8]) {
  if constexpr (VEC) {
    if (valid > 0) {
      load_n<8>(p, v);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = 0.f;
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = j < valid ? to_f(p[j]) : 0.f;
  }
}
template <typename T, bool VEC>
__device__ __forceinline__ void store8(T* p, int valid, const float (&v)[8]) {
  if constexpr (VEC) {
    if (valid > 0) store_n<8>(p, v);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (j < valid) p[j] = from_f<T>(v[j]);
  }
}

// y (may be null) = gelu(x); q, e (may be null) = x in 8 bits
template <typename T, bool VEC, bool GELU, bool PACK>
__global__ __launch_bounds__(kThreads)
void act8_fwd_kernel(const T* __restrict__ x, T* __restrict__ y,
                     int8_t* __restrict__ q, uint8_t* __restrict__ e,
                     long long chunks, long long nb, long long dim) {
  const long long step = (long long)gridDim.x * kThreads;
  // chunks is a multiple of 16: a block's 16 lanes stay together
  for (long long c = (long long)blockIdx.x * kThreads + threadIdx.x;
       c < chunks; c += step) {
    const Chunk k = chunk_at(c, nb);
    const long long at = k.row * dim + k.col;
    const int valid = (int)(dim - k.col < 8 ? dim - k.col : 8);
    float v[8];
    load8<T, VEC>(x + at, valid, v);
    if constexpr (PACK) {
      uint32_t ex;
      u32x2 w;
      pack8(v, ex, w);
      if (k.sub == 0) e[k.blk] = (uint8_t)ex;
      if constexpr (VEC) {
        if (valid > 0) *reinterpret_cast<u32x2*>(q + at) = w;
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (j < valid) q[at + j] = (int8_t)(w[j >> 2] >> (8 * (j & 3)));
      }
    }
    if constexpr (GELU) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        float ex2;
        v[j] *= normal_cdf<T>(v[j], ex2);
      }
      store8<T, VEC>(y + at, valid, v);
    }
  }
}

template <typename T, bool VEC>
__global__ __launch_bounds__(kThreads)
void gelu_bwd_kernel(const T* __restrict__ dy, const int8_t* __restrict__ q,
                     const uint8_t* __restrict__ e, T* __restrict__ dx,
                     long long chunks, long long nb, long long dim) {
  const long long step = (long long)gridDim.x * kThreads;
  for (long long c = (long long)blockIdx.x * kThreads + threadIdx.x;
       c < chunks; c += step) {
    const Chunk k = chunk_at(c, nb);
    const long long at = k.row * dim + k.col;
    const int valid = (int)(dim - k.col < 8 ? dim - k.col : 8);
    const float unit = __uint_as_float((uint32_t)e[k.blk] << 23);
    float d[8], v[8];
    load8<T, VEC>(dy + at, valid, d);
    if constexpr (VEC) {
      u32x2 w = {0u, 0u};
      if (valid > 0) w = *reinterpret_cast<const u32x2*>(q + at);
#pragma unroll
      for (int j = 0; j < 8; ++j)
        v[j] = (float)(int8_t)(w[j >> 2] >> (8 * (j & 3))) * unit;
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        v[j] = j < valid ? (float)q[at + j] * unit : 0.f;
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      float ex;
      const float cdf = normal_cdf<T>(v[j], ex);
      d[j] *= fmaf(v[j] * ex, 0.3989422804014327f, cdf);
    }
    store8<T, VEC>(dx + at, valid, d);
  }
}

bool aligned(const void* p, int n) {
  return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0;
}
unsigned chunk_grid(long long chunks) {
  return (unsigned)std::min<long long>(ceil_div(chunks, kThreads), 1 << 22);
}

template <typename T>
void fwd_t(const T* x, T* y, int8_t* q, uint8_t* e, long long rows,
           long long dim, hipStream_t s) {
  const long long nb = ceil_div(dim, 128), chunks = rows * nb * 16;
  const bool vec = dim % 8 == 0 && aligned(x, 16) && (!y || aligned(y, 16))
      && (!q || aligned(q, 8));
  const unsigned grid = chunk_grid(chunks);
#define BLADES_FWD(V, G, P)                                             \
  act8_fwd_kernel<T, V, G, P>                                           \
      <<<grid, kThreads, 0, s>>>(x, y, q, e, chunks, nb, dim)
  if (vec) {
    if (y && q) BLADES_FWD(true, true, true);
    else if (y) BLADES_FWD(true, true, false);
    else BLADES_FWD(true, false, true);
  } else {
    if (y && q) BLADES_FWD(false, true, true);
    else if (y) BLADES_FWD(false, true, false);
    else BLADES_FWD(false, false, true);
  }
#undef BLADES_FWD
}

template <typename T>
void bwd_t(const T* dy, const int8_t* q, const uint8_t* e, T* dx,
           long long rows, long long dim, hipStream_t s) {
  const long long nb = ceil_div(dim, 128), chunks = rows * nb * 16;
  const bool vec = dim % 8 == 0 && aligned(dy, 16) && aligned(dx, 16)
      && aligned(q, 8);
  const unsigned grid = chunk_grid(chunks);
  if (vec)
    gelu_bwd_kernel<T, true>
        <<<grid, kThreads, 0, s>>>(dy, q, e, dx, chunks, nb, dim);
  else
    gelu_bwd_kernel<T, false>
        <<<grid, kThreads, 0, s>>>(dy, q, e, dx, chunks, nb, dim);
}

}  // namespace

void act8_pack(const void* x, int8_t* q, uint8_t* e, long long rows,
               long long dim, DType t, hipStream_t s) {
  gelu_forward(x, nullptr, q, e, rows, dim, t, s);
}

void gelu_forward(const void* x, void* y, int8_t* q, uint8_t* e,
                  long long rows, long long dim, DType t, hipStream_t s) {
  if (t == kF32)
    fwd_t(static_cast<const float*>(x), static_cast<float*>(y), q, e, rows,
          dim, s);
  else
    fwd_t(static_cast<const bf16*>(x), static_cast<bf16*>(y), q, e, rows, dim,
          s);
}

void gelu_backward(const void* dy, const int8_t* q, const uint8_t* e,
                   void* dx, long long rows, long long dim, DType t,
                   hipStream_t s) {
  if (t == kF32)
    bwd_t(static_cast<const float*>(dy), q, e, static_cast<float*>(dx), rows,
          dim, s);
  else
    bwd_t(static_cast<const bf16*>(dy), q, e, static_cast<bf16*>(dx), rows,
          dim, s);
}

}  // namespace token_ops
