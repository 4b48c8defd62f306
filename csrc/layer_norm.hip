// Layer norm, forward and backward, for a population of clients.
//
//   y  = (x - mean) * rstd * w + b,   rstd = 1 / sqrt(var + eps)
//   g  = dy * w,  h = (x - mean) * rstd
//   dx = rstd * (g - mean(g) - h * mean(g * h))
//   dw = sum_rows dy * h,   db = sum_rows dy     (per client)
//
// Bound by memory: forward moves 2, backward 3 elements per value.  A row
// stays in the registers of 16, 64 or 256 threads from its one read to its
// one write, so statistics are taken in two steps (mean, then centred
// squares) at no traffic.  The backward block walks rows of one client and
// keeps its columns' dw and db in registers; blocks leave one partial row
// each, summed in a fixed order by a second kernel: no atomics, so results
// repeat bit for bit.  Rows wider than the registers hold (or wide rows
// without 16-byte alignment) take kernels that read the row again instead.
// Measured: 16383 x 4096 bf16 forward 62 us (4.3 TB/s), backward 82 us
// (4.9 TB/s, 7 us more to join); 204800 x 128 fp32 in 100 clients 37 and
// 59 us.  One value an access costs: 16383 x 2047 bf16 67 and 61 us against 27
// and 51 for 2048, 16383 x 4095 bf16, in the kernels that read again, 159 and
// 248 against 54 and 92 (fp32: 273 and 342 against 98 and 161).

#include "token_ops.h"
#include "token_device.h"

#include <algorithm>

namespace token_ops {
namespace {

constexpr int kThreads = 256;

// Sum over the TPR threads of a row.  For TPR == 256 `red` holds one slot per
// wave and value.  There is one barrier, between writing and reading it: calls
// take turns with two such arrays, so that the other one's barrier lies
// between reading an array and writing it again.
template <int TPR, int N>
__device__ __forceinline__ void row_sum(float (&v)[N], float* red) {
  constexpr int W = TPR < 64 ? TPR : 64;
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = lanes_sum<W>(v[i]);
  if constexpr (TPR > 64) {
    const int wave = threadIdx.x >> 6;
    if ((threadIdx.x & 63) == 0) {
#pragma unroll
      for (int i = 0; i < N; ++i) red[wave * N + i] = v[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) {
      float s = 0.f;
#pragma unroll
      for (int w = 0; w < TPR / 64; ++w) s += red[w * N + i];
      v[i] = s;
    }
  }
}

// VEC values as they lie in memory
template <typename T, int VEC> struct Packed { T v[VEC]; };
template <> struct Packed<float, 4> { f32x4 v; };
template <> struct Packed<bf16, 8> { u32x4 v; };

template <typename T, int VEC>
__device__ __forceinline__ void fetch(const T* p, Packed<T, VEC>& r) {
  if constexpr (VEC == Vec16<T>::n) {
    r.v = *reinterpret_cast<const decltype(r.v)*>(p);
  } else {
#pragma unroll
    for (int j = 0; j < VEC; ++j) r.v[j] = p[j];
  }
}
template <int VEC>
__device__ __forceinline__ void unpack(const Packed<float, VEC>& r,
                                       float (&v)[VEC]) {
#pragma unroll
  for (int j = 0; j < VEC; ++j) v[j] = r.v[j];
}
template <int VEC>
__device__ __forceinline__ void unpack(const Packed<bf16, VEC>& r,
                                       float (&v)[VEC]) {
  if constexpr (VEC == 8) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      v[2 * j] = __uint_as_float(r.v[j] << 16);
      v[2 * j + 1] = __uint_as_float(r.v[j] & 0xffff0000u);
    }
  } else {
#pragma unroll
    for (int j = 0; j < VEC; ++j) v[j] = (float)r.v[j];
  }
}

template <typename T, int VEC, int NV, int TPR>
__global__ __launch_bounds__(kThreads)
void norm_fwd_kernel(NormArgs a) {
  constexpr int RPB = kThreads / TPR;
  __shared__ float red[2][8];
  const int lane = threadIdx.x % TPR;
  const long long total = a.groups * a.rows;
  const int dim = (int)a.dim;
  // a row slot's threads leave the loop together, a block's for TPR == 256
  for (long long row = (long long)blockIdx.x * RPB + threadIdx.x / TPR;
       row < total; row += (long long)gridDim.x * RPB) {
    const long long g = a.groups == 1 ? 0 : row / a.rows;
    const T* x = static_cast<const T*>(a.x) + row * a.dim;

    float v[NV][VEC];
    float s[2] = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * TPR + lane) * VEC;
      if (c < dim) {
        load_n<VEC>(x + c, v[i]);
      } else {
#pragma unroll
        for (int j = 0; j < VEC; ++j) v[i][j] = 0.f;
      }
#pragma unroll
      for (int j = 0; j < VEC; ++j) s[0] += v[i][j];
    }
    float one[1] = {s[0]};
    row_sum<TPR, 1>(one, red[0]);
    const float inv = 1.f / (float)dim;
    float mean = one[0] * inv;
    // The centred values' own mean corrects what the first sum rounded away,
    // which matters where the mean is large against the deviation.
    s[0] = s[1] = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * TPR + lane) * VEC;
      if (c < dim) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          const float d = v[i][j] - mean;
          s[0] += d;
          s[1] += d * d;
        }
      }
    }
    row_sum<TPR, 2>(s, red[1]);
    const float off = s[0] * inv;
    const float rstd = 1.f / sqrtf(fmaxf(s[1] * inv - off * off, 0.f) + a.eps);
    mean += off;

    const T* w = a.w ? static_cast<const T*>(a.w) + g * a.w_stride : nullptr;
    const T* b = a.b ? static_cast<const T*>(a.b) + g * a.b_stride : nullptr;
    T* y = static_cast<T*>(a.y) + row * a.dim;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * TPR + lane) * VEC;
      if (c < dim) {
        float wv[VEC], bv[VEC];
        if (w) load_n<VEC>(w + c, wv);
        if (b) load_n<VEC>(b + c, bv);
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          float h = (v[i][j] - mean) * rstd;
          if (w) h *= wv[j];
          if (b) h += bv[j];
          v[i][j] = h;
        }
        store_n<VEC>(y + c, v[i]);
      }
    }
    if (lane == 0) {
      a.mean[row] = mean;
      a.rstd[row] = rstd;
    }
  }
}

// grid (blocks per group, groups); partial[g][block][2][dim]
template <typename T, int VEC, int NV, int TPR, bool PARAMS>
__global__ __launch_bounds__(kThreads)
void norm_bwd_kernel(NormArgs a) {
  constexpr int RPB = kThreads / TPR;
  constexpr int SPAN = TPR * VEC * NV;            // columns a row slot holds
  __shared__ float red[2][8];
  __shared__ float comb[PARAMS && TPR <= 64 ? 4 * SPAN : 1];
  const int lane = threadIdx.x % TPR;
  const int dim = (int)a.dim;
  const long long g = blockIdx.y;
  const long long base = g * a.rows;
  const T* wp = a.w ? static_cast<const T*>(a.w) + g * a.w_stride : nullptr;
  const float inv = 1.f / (float)dim;

  float w[NV][VEC];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = (i * TPR + lane) * VEC;
    if (wp && c < dim) {
      load_n<VEC>(wp + c, w[i]);
    } else {
#pragma unroll
      for (int j = 0; j < VEC; ++j) w[i][j] = 1.f;
    }
  }
  float dw[NV][VEC], db[NV][VEC];
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int j = 0; j < VEC; ++j) dw[i][j] = db[i][j] = 0.f;

  // The next row's values are fetched while this one's are reduced, where
  // registers allow (16383 x 4096 bf16: 82 us against 99; the forward pass,
  // whose blocks are many and short, gains nothing from it: 65 against 62).
  constexpr bool AHEAD = NV * VEC <= 32;
  const long long step = (long long)gridDim.x * RPB;
  Packed<T, VEC> px[NV], pd[NV];
  float pm = 0.f, pr = 0.f;
  auto fetch_row = [&](long long r0) {
    const long long r = r0 + threadIdx.x / TPR;
    if (r < a.rows) {                             // uniform over a row slot
      const long long row = base + r;
      pm = a.mean[row];
      pr = a.rstd[row];
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int c = (i * TPR + lane) * VEC;
        if (c < dim) {
          fetch<T, VEC>(static_cast<const T*>(a.x) + row * a.dim + c, px[i]);
          fetch<T, VEC>(static_cast<const T*>(a.dy) + row * a.dim + c, pd[i]);
        }
      }
    }
  };
  int turn = 0;
  if (AHEAD) fetch_row((long long)blockIdx.x * RPB);
  for (long long r0 = (long long)blockIdx.x * RPB; r0 < a.rows;
       r0 += step, turn ^= 1) {
    const long long r = r0 + threadIdx.x / TPR;
    const bool live = r < a.rows;                 // uniform over a row slot
    const long long row = base + (live ? r : 0);
    if (!AHEAD) fetch_row(r0);
    const float mean = pm, rstd = pr;
    float h[NV][VEC], d[NV][VEC];
    float s[2] = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      unpack(px[i], h[i]);
      unpack(pd[i], d[i]);
    }
    if (AHEAD) fetch_row(r0 + step);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * TPR + lane) * VEC;
      if (live && c < dim) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          h[i][j] = (h[i][j] - mean) * rstd;
          if (PARAMS) {
            dw[i][j] += d[i][j] * h[i][j];
            db[i][j] += d[i][j];
          }
          d[i][j] *= w[i][j];
          s[0] += d[i][j];
          s[1] += d[i][j] * h[i][j];
        }
      }
    }
    row_sum<TPR, 2>(s, red[turn]);
    const float c1 = s[0] * inv, c2 = s[1] * inv;
    T* dx = static_cast<T*>(a.y) + row * a.dim;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * TPR + lane) * VEC;
      if (live && c < dim) {
#pragma unroll
        for (int j = 0; j < VEC; ++j)
          d[i][j] = rstd * (d[i][j] - c1 - h[i][j] * c2);
        store_n<VEC>(dx + c, d[i]);
      }
    }
  }

  if constexpr (PARAMS) {
    float* out = a.partial
        + ((g * gridDim.x + blockIdx.x) * 2) * a.dim;
    if constexpr (TPR <= 64) {
      const int wave = threadIdx.x >> 6;
#pragma unroll
      for (int which = 0; which < 2; ++which) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
#pragma unroll
          for (int j = 0; j < VEC; ++j) {
            float v = which ? db[i][j] : dw[i][j];
#pragma unroll
            for (int o = TPR; o < 64; o <<= 1) v += __shfl_xor(v, o, 64);
            if ((threadIdx.x & 63) < TPR)
              comb[wave * SPAN + (i * TPR + lane) * VEC + j] = v;
          }
        }
        __syncthreads();
        for (int c = threadIdx.x; c < dim; c += kThreads)
          out[which * a.dim + c] = (comb[c] + comb[SPAN + c])
              + (comb[2 * SPAN + c] + comb[3 * SPAN + c]);
        __syncthreads();
      }
    } else {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int c = (i * TPR + lane) * VEC;
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          if (c + j < dim) {
            out[c + j] = dw[i][j];
            out[a.dim + c + j] = db[i][j];
          }
        }
      }
    }
  }
}

// Any width: one block per row, the row read three times (the second and
// third come from the caches).
template <typename T>
__global__ __launch_bounds__(kThreads)
void norm_fwd_wide_kernel(NormArgs a) {
  __shared__ float red[2][8];
  for (long long row = blockIdx.x; row < a.groups * a.rows;
       row += gridDim.x) {
    const long long g = row / a.rows;
    const T* x = static_cast<const T*>(a.x) + row * a.dim;
    const float inv = 1.f / (float)a.dim;
    float one[1] = {0.f};
    for (long long c = threadIdx.x; c < a.dim; c += kThreads)
      one[0] += to_f(x[c]);
    row_sum<256, 1>(one, red[0]);
    float mean = one[0] * inv;
    float s[2] = {0.f, 0.f};
    for (long long c = threadIdx.x; c < a.dim; c += kThreads) {
      const float d = to_f(x[c]) - mean;
      s[0] += d;
      s[1] += d * d;
    }
    row_sum<256, 2>(s, red[1]);
    const float off = s[0] * inv;
    const float rstd = 1.f / sqrtf(fmaxf(s[1] * inv - off * off, 0.f) + a.eps);
    mean += off;
    const T* w = a.w ? static_cast<const T*>(a.w) + g * a.w_stride : nullptr;
    const T* b = a.b ? static_cast<const T*>(a.b) + g * a.b_stride : nullptr;
    T* y = static_cast<T*>(a.y) + row * a.dim;
    for (long long c = threadIdx.x; c < a.dim; c += kThreads) {
      float h = (to_f(x[c]) - mean) * rstd;
      if (w) h *= to_f(w[c]);
      if (b) h += to_f(b[c]);
      y[c] = from_f<T>(h);
    }
    if (threadIdx.x == 0) { a.mean[row] = mean; a.rstd[row] = rstd; }
  }
}

template <typename T>
__global__ __launch_bounds__(kThreads)
void norm_bwd_wide_kernel(NormArgs a) {
  __shared__ float red[2][8];
  int turn = 0;
  for (long long row = blockIdx.x; row < a.groups * a.rows;
       row += gridDim.x, turn ^= 1) {
    const long long g = row / a.rows;
    const T* x = static_cast<const T*>(a.x) + row * a.dim;
    const T* dy = static_cast<const T*>(a.dy) + row * a.dim;
    const T* w = a.w ? static_cast<const T*>(a.w) + g * a.w_stride : nullptr;
    T* dx = static_cast<T*>(a.y) + row * a.dim;
    const float mean = a.mean[row], rstd = a.rstd[row];
    float s[2] = {0.f, 0.f};
    for (long long c = threadIdx.x; c < a.dim; c += kThreads) {
      const float h = (to_f(x[c]) - mean) * rstd;
      const float d = to_f(dy[c]) * (w ? to_f(w[c]) : 1.f);
      s[0] += d;
      s[1] += d * h;
    }
    row_sum<256, 2>(s, red[turn]);
    const float inv = 1.f / (float)a.dim;
    const float c1 = s[0] * inv, c2 = s[1] * inv;
    for (long long c = threadIdx.x; c < a.dim; c += kThreads) {
      const float h = (to_f(x[c]) - mean) * rstd;
      const float d = to_f(dy[c]) * (w ? to_f(w[c]) : 1.f);
      dx[c] = from_f<T>(rstd * (d - c1 - h * c2));
    }
  }
}

// dw and db of wide rows: a thread owns a column and walks the block's rows.
// grid (column blocks, row blocks, groups)
template <typename T>
__global__ __launch_bounds__(kThreads)
void norm_params_wide_kernel(NormArgs a) {
  const long long c = (long long)blockIdx.x * kThreads + threadIdx.x;
  if (c >= a.dim) return;
  const long long g = blockIdx.z;
  float dw = 0.f, db = 0.f;
  for (long long r = blockIdx.y; r < a.rows; r += gridDim.y) {
    const long long row = g * a.rows + r;
    const float d = to_f(static_cast<const T*>(a.dy)[row * a.dim + c]);
    const float h = (to_f(static_cast<const T*>(a.x)[row * a.dim + c])
                     - a.mean[row]) * a.rstd[row];
    dw += d * h;
    db += d;
  }
  float* out = a.partial + ((g * gridDim.y + blockIdx.y) * 2) * a.dim;
  out[c] = dw;
  out[a.dim + c] = db;
}

// Sums `blocks` partial rows of `width` floats per group.  A block takes 32
// columns at a time; its 8 row lanes walk the partials and meet in shared
// memory.
// Columns below `split` go to out0, the rest to out1 (either may be null).
template <typename T>
__global__ __launch_bounds__(kThreads)
void join_rows_kernel(const float* __restrict__ partial, long long blocks,
                      long long width, long long split, T* out0,
                      long long out0_group, T* out1, Scale scale) {
  __shared__ float part[8][33];
  const int cl = threadIdx.x & 31, rl = threadIdx.x >> 5;
  const long long g = blockIdx.y;
  const float* p = partial + g * blocks * width;
  for (long long c0 = (long long)blockIdx.x * 32; c0 < width;
       c0 += (long long)gridDim.x * 32) {
    const long long c = c0 + cl;
    float s = 0.f;
    if (c < width) {
      float s1 = 0.f, s2 = 0.f, s3 = 0.f;
      long long r = rl;
      for (; r + 24 < blocks; r += 32) {
        s += p[r * width + c];
        s1 += p[(r + 8) * width + c];
        s2 += p[(r + 16) * width + c];
        s3 += p[(r + 24) * width + c];
      }
      for (; r < blocks; r += 8) s += p[r * width + c];
      s = (s + s1) + (s2 + s3);
    }
    part[rl][cl] = s;
    __syncthreads();
    if (rl == 0 && c < width) {
#pragma unroll
      for (int i = 1; i < 8; ++i) s += part[i][cl];
      s = scaled(s, scale_of(scale, g));
      if (c < split) {
        if (out0) out0[g * out0_group + c] = from_f<T>(s);
      } else if (out1) {
        out1[g * (width - split) + (c - split)] = from_f<T>(s);
      }
    }
    __syncthreads();
  }
}

template <typename T, int VEC>
__global__ __launch_bounds__(kThreads)
void colsum_kernel(const T* __restrict__ x, float* __restrict__ partial,
                   long long rows, long long cols) {
  // 32 column vectors x 8 row lanes per block
  __shared__ float part[8][32 * VEC];
  const int cl = threadIdx.x & 31, rl = threadIdx.x >> 5;
  const long long c = ((long long)blockIdx.x * 32 + cl) * VEC;
  const long long g = blockIdx.z;
  const T* p = x + g * rows * cols;
  float s[VEC];
#pragma unroll
  for (int j = 0; j < VEC; ++j) s[j] = 0.f;
  if (c < cols) {
    const long long step = 8ll * gridDim.y;
#pragma unroll 4
    for (long long r = blockIdx.y * 8ll + rl; r < rows; r += step) {
      float v[VEC];
      load_n<VEC>(p + r * cols + c, v);
#pragma unroll
      for (int j = 0; j < VEC; ++j) s[j] += v[j];
    }
  }
#pragma unroll
  for (int j = 0; j < VEC; ++j) part[rl][cl * VEC + j] = s[j];
  __syncthreads();
  float* out = partial + (g * gridDim.y + blockIdx.y) * cols;
  const long long c0 = (long long)blockIdx.x * 32 * VEC;
  for (int i = threadIdx.x; i < 32 * VEC; i += kThreads) {
    if (c0 + i < cols) {
      float t = 0.f;
#pragma unroll
      for (int k = 0; k < 8; ++k) t += part[k][i];
      out[c0 + i] = t;
    }
  }
}

// A launch may hold 2^32 threads; kernels stride over what is beyond.
unsigned row_grid(long long blocks) {
  return (unsigned)std::min<long long>(blocks, 1 << 22);
}

bool aligned16(const void* p) {
  return (reinterpret_cast<uintptr_t>(p) & 15) == 0;
}

// Threads per row and vectors per thread for `units` vectors a row:
// index into {16x1, 16x2, 64x1, 64x2, 64x4, 256x2, 256x4, 256x8}, -1: wide.
int norm_shape(long long units) {
  const long long cap[8] = {16, 32, 64, 128, 256, 512, 1024, 2048};
  for (int i = 0; i < 8; ++i)
    if (units <= cap[i]) return i;
  return -1;
}
const int kTpr[8] = {16, 16, 64, 64, 64, 256, 256, 256};

template <typename T, int VEC, int NV, int TPR>
void launch_fwd(const NormArgs& a, hipStream_t s) {
  const long long blocks = ceil_div(a.groups * a.rows, kThreads / TPR);
  norm_fwd_kernel<T, VEC, NV, TPR>
      <<<row_grid(blocks), kThreads, 0, s>>>(a);
}

template <typename T, int VEC, int NV, int TPR>
void launch_bwd(const NormArgs& a, long long blocks, hipStream_t s) {
  const dim3 grid((unsigned)blocks, (unsigned)a.groups);
  if (a.partial)
    norm_bwd_kernel<T, VEC, NV, TPR, true><<<grid, kThreads, 0, s>>>(a);
  else
    norm_bwd_kernel<T, VEC, NV, TPR, false><<<grid, kThreads, 0, s>>>(a);
}

template <typename T, int VEC>
bool fwd_shape(const NormArgs& a, hipStream_t s) {
  switch (norm_shape(ceil_div(a.dim, VEC))) {
    case 0: launch_fwd<T, VEC, 1, 16>(a, s); return true;
    case 1: launch_fwd<T, VEC, 2, 16>(a, s); return true;
    case 2: launch_fwd<T, VEC, 1, 64>(a, s); return true;
    case 3: launch_fwd<T, VEC, 2, 64>(a, s); return true;
    case 4: launch_fwd<T, VEC, 4, 64>(a, s); return true;
    case 5: launch_fwd<T, VEC, 2, 256>(a, s); return true;
    case 6: launch_fwd<T, VEC, 4, 256>(a, s); return true;
    case 7: launch_fwd<T, VEC, 8, 256>(a, s); return true;
  }
  return false;
}

template <typename T, int VEC>
bool bwd_shape(const NormArgs& a, long long blocks, hipStream_t s) {
  switch (norm_shape(ceil_div(a.dim, VEC))) {
    case 0: launch_bwd<T, VEC, 1, 16>(a, blocks, s); return true;
    case 1: launch_bwd<T, VEC, 2, 16>(a, blocks, s); return true;
    case 2: launch_bwd<T, VEC, 1, 64>(a, blocks, s); return true;
    case 3: launch_bwd<T, VEC, 2, 64>(a, blocks, s); return true;
    case 4: launch_bwd<T, VEC, 4, 64>(a, blocks, s); return true;
    case 5: launch_bwd<T, VEC, 2, 256>(a, blocks, s); return true;
    case 6: launch_bwd<T, VEC, 4, 256>(a, blocks, s); return true;
    case 7: launch_bwd<T, VEC, 8, 256>(a, blocks, s); return true;
  }
  return false;
}

template <typename T>
bool vector_ok(const NormArgs& a) {
  constexpr int V = Vec16<T>::n;
  return a.dim % V == 0 && aligned16(a.x) && aligned16(a.y)
      && (!a.dy || aligned16(a.dy)) && (!a.w || aligned16(a.w))
      && (!a.b || aligned16(a.b));
}

template <typename T>
void forward_t(const NormArgs& a, hipStream_t s) {
  const bool done = vector_ok<T>(a) ? fwd_shape<T, Vec16<T>::n>(a, s)
                                    : fwd_shape<T, 1>(a, s);
  if (!done)
    norm_fwd_wide_kernel<T>
        <<<row_grid(a.groups * a.rows), kThreads, 0, s>>>(a);
}

template <typename T>
void backward_t(const NormArgs& a, hipStream_t s) {
  const DType t = sizeof(T) == 4 ? kF32 : kBF16;
  const long long blocks = norm_partial_blocks(a.groups, a.rows, a.dim, t);
  const bool done = vector_ok<T>(a) ? bwd_shape<T, Vec16<T>::n>(a, blocks, s)
                                    : bwd_shape<T, 1>(a, blocks, s);
  if (!done) {
    norm_bwd_wide_kernel<T>
        <<<row_grid(a.groups * a.rows), kThreads, 0, s>>>(a);
    if (a.partial)
      norm_params_wide_kernel<T>
          <<<dim3((unsigned)ceil_div(a.dim, kThreads), (unsigned)blocks,
                  (unsigned)a.groups), kThreads, 0, s>>>(a);
  }
  if (a.partial)
    join_rows_kernel<T>
        <<<dim3(row_grid(ceil_div(2 * a.dim, 32)), (unsigned)a.groups),
           kThreads, 0, s>>>(a.partial, blocks, 2 * a.dim, a.dim,
                             static_cast<T*>(a.dw), a.dim,
                             static_cast<T*>(a.db), Scale{});
}

}  // namespace

// Blocks per group of the backward kernel.  About 1024 in all (4 per compute
// unit) keep the chip full; blocks that own a whole wide row are as fast with
// 512, and leave half the partial rows to join (16383 x 4096 bf16: 82 + 7 us
// against 94 + 11).
long long norm_partial_blocks(long long groups, long long rows, long long dim,
                              DType t) {
  const int vec = t == kF32 ? 4 : 8;
  const int shape = norm_shape(ceil_div(dim, dim % vec ? 1 : vec));
  const long long rpb = shape < 0 ? 1 : kThreads / kTpr[shape];
  const long long want =
      std::max<long long>(1, ceil_div(rpb == 1 ? 512 : 1024, groups));
  return std::max<long long>(1, std::min(want, ceil_div(rows, rpb)));
}

void norm_forward(const NormArgs& a, DType t, hipStream_t s) {
  if (t == kF32) forward_t<float>(a, s); else forward_t<bf16>(a, s);
}

void norm_backward(const NormArgs& a, DType t, hipStream_t s) {
  if (t == kF32) backward_t<float>(a, s); else backward_t<bf16>(a, s);
}

long long colsum_blocks(long long groups, long long rows, long long cols) {
  const long long per = ceil_div(cols, 128) * groups;
  const long long want = std::max<long long>(1, ceil_div(1024, per));
  return std::max<long long>(1, std::min(want, ceil_div(rows, 32)));
}

void colsum(const void* x, void* out, float* partial, long long groups,
            long long rows, long long cols, DType t, hipStream_t s) {
  const long long blocks = colsum_blocks(groups, rows, cols);
  const bool wide = cols % 4 == 0 && (t == kF32 || cols % 8 == 0)
      && aligned16(x);
  const int vec = !wide ? 1 : t == kF32 ? 4 : 8;
  const dim3 grid((unsigned)ceil_div(cols, 32 * vec), (unsigned)blocks,
                  (unsigned)groups);
  if (t == kF32) {
    const float* p = static_cast<const float*>(x);
    if (wide)
      colsum_kernel<float, 4><<<grid, kThreads, 0, s>>>(p, partial, rows, cols);
    else
      colsum_kernel<float, 1><<<grid, kThreads, 0, s>>>(p, partial, rows, cols);
  } else {
    const bf16* p = static_cast<const bf16*>(x);
    if (wide)
      colsum_kernel<bf16, 8><<<grid, kThreads, 0, s>>>(p, partial, rows, cols);
    else
      colsum_kernel<bf16, 1><<<grid, kThreads, 0, s>>>(p, partial, rows, cols);
  }
  join_rows(partial, groups, blocks, cols, out, cols, Scale{}, t, s);
}

void join_rows(const float* partial, long long groups, long long blocks,
               long long cols, void* out, long long out_group,
               const Scale& scale, DType t, hipStream_t s) {
  const dim3 grid(row_grid(ceil_div(cols, 32)), (unsigned)groups);
  if (t == kF32)
    join_rows_kernel<float><<<grid, kThreads, 0, s>>>(
        partial, blocks, cols, cols, static_cast<float*>(out), out_group,
        nullptr, scale);
  else
    join_rows_kernel<bf16><<<grid, kThreads, 0, s>>>(
        partial, blocks, cols, cols, static_cast<bf16*>(out), out_group,
        nullptr, scale);
}

}  // namespace token_ops
