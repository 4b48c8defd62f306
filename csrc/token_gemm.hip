// Matrix products on the matrix cores for the linear layers of token models,
// with the epilogues of a large-vocabulary loss.
//
// One tile loop serves every product; operands differ in
//   * type: bf16 as it is; fp32 cut into three bf16 parts; 8-bit activations
//     (act8.hip), whose stored values are exact in bf16;
//   * order: contraction along the rows ([m][k]) or across them ([k][m]).
//
// fp32: x = hi + mid + lo by truncation is exact (8 + 8 + 8 bits), and the
// six products hi*hi, hi*mid, mid*hi, hi*lo, mid*mid, lo*hi leave out only
// terms below 2^-23 of |a||b|, so results are fp32's; six bf16 products per
// multiplication have 2.6 times the rate of the fp32 matrix instruction.
// A value that is not finite makes its results NaN (inf - inf in the parts).
//
// A block of 4 waves owns 128 x 128 of the output, each wave 64 x 64 in
// v_mfma_f32_32x32x16_bf16 tiles.  Global loads of the next step are in
// flight, in registers, while the current step multiplies out of LDS.
//   [m][k] tiles lie in LDS as [128][BK] with 16-byte columns swizzled by the
//   row: the 16-byte fragment reads touch every bank once.
//   [k][m] tiles lie as [BK][128] and are read by ds_read_b64_tr_b16, which
//   hands each lane 4 values down a column; 32-byte columns swizzled by k.
// Sums are 32-bit in the accumulators.

#include "token_ops.h"
#include "token_device.h"

#include <algorithm>

namespace token_ops {
namespace {

constexpr int kThreads = 256;
constexpr int kTile = 128;

enum Src { F32, BF16, ACT8 };
enum Epi { STORE, LSE, GRAD };

template <Src S> struct SrcOf;
template <> struct SrcOf<F32> { using T = float; static constexpr int P = 3; };
template <> struct SrcOf<BF16> { using T = bf16; static constexpr int P = 1; };
template <> struct SrcOf<ACT8> { using T = int8_t; static constexpr int P = 1; };

// What a kernel knows of an operand: `rows` of the output it feeds (m or n),
// and how far the contiguous axis may be read.
struct Op {
  const void* p;
  long long ld, group;
  long long rows, ext;
  const uint8_t* e;
  long long e_ld, e_group;
};

struct Params {
  Op a, b;
  long long k;
  int tiles_m, tiles_n, splits;
  // STORE
  void* out;
  long long out_ld, out_group;
  int out_f32, accumulate;
  const void* bias;
  long long bias_group;
  float* partial;
  // LSE, GRAD: m runs over the vocabulary, n over the tokens
  const long long* target;
  long long ignore, v0;
  float2* part;
  float* picked;
  const float* lse;
  const float* grad;
  long long grad_g, grad_n;
  const float* count;
};

// Three bf16 parts of 8 floats, packed in pairs.
__device__ __forceinline__ void split3(const float (&x)[8], u32x4 (&o)[3]) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    uint32_t h[2], m[2], l[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const float v = x[2 * j + i];
      h[i] = __float_as_uint(v);
      const float r = v - __uint_as_float(h[i] & 0xffff0000u);
      m[i] = __float_as_uint(r);
      l[i] = __float_as_uint(r - __uint_as_float(m[i] & 0xffff0000u));
    }
    o[0][j] = __builtin_amdgcn_perm(h[1], h[0], 0x07060302u);
    o[1][j] = __builtin_amdgcn_perm(m[1], m[0], 0x07060302u);
    o[2][j] = __builtin_amdgcn_perm(l[1], l[0], 0x07060302u);
  }
}

template <Src S> struct Raw { u32x4 v; };
template <> struct Raw<F32> { float v[8]; };
template <> struct Raw<ACT8> { u32x2 v; uint32_t e; };

// Moves one operand's 128 x BK tile: global -> registers -> LDS.
template <Src S, bool KM, bool VEC, int BK>
struct Loader {
  using T = typename SrcOf<S>::T;
  static constexpr int P = SrcOf<S>::P;
  static constexpr int N = kTile * BK / 8 / kThreads;   // chunks a thread
  static constexpr int PLANE = kTile * BK;              // bf16 values
  const T* p;
  const uint8_t* e;
  long long ld, e_ld;
  long long ext;       // end of the contiguous axis
  long long row0;      // first row of the tile ([m][k]) or column ([k][m])
  long long rows;
  long long kend;
  Raw<S> raw[N];

  __device__ __forceinline__ void init(const Op& o, long long g,
                                       long long tile, long long kend_) {
    p = static_cast<const T*>(o.p) + g * o.group;
    e = o.e ? o.e + g * o.e_group : nullptr;
    ld = o.ld;
    e_ld = o.e_ld;
    ext = o.ext;
    rows = o.rows;
    row0 = tile * kTile;
    kend = kend_;
  }

  // r, c: row and first column in memory; lim: columns beyond are zero
  __device__ __forceinline__ void fetch(Raw<S>& w, bool ok, long long r,
                                        long long c, long long lim) {
    const T* q = p + r * ld + c;
    if constexpr (S == F32) {
      if constexpr (VEC) {
        f32x4 x = {0, 0, 0, 0}, y = {0, 0, 0, 0};
        if (ok && c < lim) x = *reinterpret_cast<const f32x4*>(q);
        if (ok && c + 4 < lim) y = *reinterpret_cast<const f32x4*>(q + 4);
#pragma unroll
        for (int j = 0; j < 4; ++j) { w.v[j] = x[j]; w.v[4 + j] = y[j]; }
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
          w.v[j] = (ok && c + j < lim) ? q[j] : 0.f;
      }
    } else if constexpr (S == BF16) {
      w.v = u32x4{0, 0, 0, 0};
      if constexpr (VEC) {
        if (ok && c < lim) w.v = *reinterpret_cast<const u32x4*>(q);
      } else {
        const uint16_t* h = reinterpret_cast<const uint16_t*>(q);
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (ok && c + j < lim)
            w.v[j >> 1] |= (uint32_t)h[j] << (16 * (j & 1));
      }
    } else {
      w.v = u32x2{0, 0};
      w.e = 0;
      if (ok && c < lim) w.e = e[r * e_ld + (c >> 7)];
      if constexpr (VEC) {
        if (ok && c < lim) w.v = *reinterpret_cast<const u32x2*>(q);
      } else {
        const uint8_t* h = reinterpret_cast<const uint8_t*>(q);
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (ok && c + j < lim)
            w.v[j >> 2] |= (uint32_t)h[j] << (8 * (j & 3));
      }
    }
  }

  __device__ __forceinline__ void load(long long k0) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int id = i * kThreads + threadIdx.x;
      if constexpr (KM) {
        const long long k = k0 + (id >> 4);
        fetch(raw[i], k < kend, k, row0 + (id & 15) * 8, ext);
      } else {
        const long long r = row0 + id / (BK / 8);
        const long long lim = kend < ext ? kend : ext;
        fetch(raw[i], r < rows, r, k0 + (id % (BK / 8)) * 8, lim);
      }
    }
  }

  __device__ __forceinline__ void store(bf16* lds) const {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int id = i * kThreads + threadIdx.x;
      int at;
      if constexpr (KM) {
        const int k = id >> 4, c = id & 15;
        at = k * kTile + (((c >> 1) ^ (2 * (k & 3))) << 4) + (c & 1) * 8;
      } else {
        constexpr int CH = BK / 8;
        const int r = id / CH, c = id % CH;
        const int sw = CH == 8 ? (r & 7) : ((r >> 1) & 3);
        at = r * BK + ((c ^ sw) << 3);
      }
      u32x4 o[3];
      if constexpr (S == F32) {
        split3(raw[i].v, o);
      } else if constexpr (S == BF16) {
        o[0] = raw[i].v;
      } else {
        const float unit = __uint_as_float(raw[i].e << 23);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          float v[2];
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            const int b = 2 * j + t;
            v[t] = (float)(int8_t)(raw[i].v[b >> 2] >> (8 * (b & 3))) * unit;
          }
          o[0][j] = __builtin_amdgcn_perm(__float_as_uint(v[1]),
                                          __float_as_uint(v[0]), 0x07060302u);
        }
      }
#pragma unroll
      for (int q = 0; q < P; ++q)
        *reinterpret_cast<u32x4*>(lds + q * PLANE + at) = o[q];
    }
  }

  // Fragment of the 32 rows from `base`, contraction step ks of 16.
  static __device__ __forceinline__ bf16x8 frag(const bf16* lds, int base,
                                                int ks) {
    const int lane = threadIdx.x & 63;
    if constexpr (KM) {
      typedef short s4 __attribute__((ext_vector_type(4)));
      const int i = lane & 15;
      const int c = (base >> 4) + ((lane >> 4) & 1);
      const int k = ks * 16 + (lane >> 5) * 8 + (i >> 2);
      // k and k + 4 have the same low bits, so the same swizzle
      const bf16* q = lds + k * kTile + ((c ^ (2 * (k & 3))) << 4)
          + (i & 3) * 4;
      union { s4 h[2]; bf16x8 v; } u;
      typedef __attribute__((address_space(3))) s4* lds_s4;
      u.h[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4)(q));
      u.h[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
          (lds_s4)(q + 4 * kTile));
      return u.v;
    } else {
      constexpr int CH = BK / 8;
      const int r = base + (lane & 31);
      const int c = ks * 2 + (lane >> 5);
      const int sw = CH == 8 ? (r & 7) : ((r >> 1) & 3);
      return *reinterpret_cast<const bf16x8*>(lds + r * BK + ((c ^ sw) << 3));
    }
  }
};

// Row of accumulator element r, for the 32 x 32 tile's lane half.
__device__ __forceinline__ int acc_row(int r, int lane) {
  return (r & 3) + 8 * (r >> 2) + 4 * (lane >> 5);
}

constexpr float kLog2e = 1.4426950408889634f;

template <Src SA, bool KMA, Src SB, bool KMB, bool VEC, Epi E>
__global__ __launch_bounds__(kThreads)
void gemm_kernel(Params p) {
  constexpr int PA = SrcOf<SA>::P, PB = SrcOf<SB>::P;
  constexpr int BK = (PA == 3 || PB == 3) ? 32 : 64;
  using LA = Loader<SA, KMA, VEC, BK>;
  using LB = Loader<SB, KMB, VEC, BK>;
  __shared__ __attribute__((aligned(16))) bf16 sa[PA * LA::PLANE];
  __shared__ __attribute__((aligned(16))) bf16 sb[PB * LB::PLANE];

  // Blocks go round robin over the 8 XCDs; give each a contiguous run of
  // tiles, ordered in bands of 8 so that neighbours share operands in its L2.
  const int total = p.tiles_m * p.tiles_n;
  int tm, tn;
  {
    const int b = blockIdx.x, q = total >> 3, r = total & 7, x = b & 7;
    const int t = x * q + (x < r ? x : r) + (b >> 3);
    const int band = 8 * p.tiles_n;
    const int first = (t / band) * 8;
    const int h = p.tiles_m - first < 8 ? p.tiles_m - first : 8;
    tm = first + (t % band) % h;
    tn = (t % band) / h;
  }
  const int split = blockIdx.y;
  const long long g = blockIdx.z;
  const long long steps = (p.k + BK - 1) / BK;
  const long long s0 = steps * split / p.splits;
  const long long s1 = steps * (split + 1) / p.splits;
  const long long kend = s1 * BK < p.k ? s1 * BK : p.k;

  LA la;
  LB lb;
  la.init(p.a, g, tm, kend);
  lb.init(p.b, g, tn, kend);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int wm = (wave >> 1) * 64, wn = (wave & 1) * 64;

  f32x16 acc[2][2];
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.f;

  if (s0 < s1) {
    la.load(s0 * BK);
    lb.load(s0 * BK);
  }
  for (long long s = s0; s < s1; ++s) {
    __syncthreads();
    la.store(sa);
    lb.store(sb);
    __syncthreads();
    if (s + 1 < s1) {
      la.load((s + 1) * BK);
      lb.load((s + 1) * BK);
    }
#pragma unroll
    for (int ks = 0; ks < BK / 16; ++ks) {
      bf16x8 fa[2][PA], fb[2][PB];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
#pragma unroll
        for (int q = 0; q < PA; ++q)
          fa[i][q] = LA::frag(sa + q * LA::PLANE, wm + i * 32, ks);
#pragma unroll
        for (int q = 0; q < PB; ++q)
          fb[i][q] = LB::frag(sb + q * LB::PLANE, wn + i * 32, ks);
      }
#pragma unroll
      for (int qa = 0; qa < PA; ++qa)
#pragma unroll
        for (int qb = 0; qb < PB; ++qb) {
          if (qa + qb > 2) continue;
#pragma unroll
          for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int j = 0; j < 2; ++j)
              acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(
                  fa[i][qa], fb[j][qb], acc[i][j], 0, 0, 0);
        }
    }
  }

  const long long m0 = (long long)tm * kTile + wm;
  const long long n0 = (long long)tn * kTile + wn;
  const long long M = p.a.rows, N = p.b.rows;

  if constexpr (E == STORE) {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const long long n = n0 + j * 32 + (lane & 31);
      if (n >= N) continue;
      float bias = 0.f;
      if (p.bias && !p.partial)
        bias = p.out_f32
            ? static_cast<const float*>(p.bias)[g * p.bias_group + n]
            : (float)static_cast<const bf16*>(p.bias)[g * p.bias_group + n];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const long long m = m0 + i * 32 + acc_row(r, lane);
          if (m >= M) continue;
          const float v = acc[i][j][r] + bias;
          if (p.partial) {
            float* o = p.partial
                + (((long long)split * gridDim.z + g) * M + m) * N + n;
            *o = p.accumulate ? *o + v : v;
          } else {
            const long long at = g * p.out_group + m * p.out_ld + n;
            if (p.out_f32)
              static_cast<float*>(p.out)[at] = v;
            else
              static_cast<bf16*>(p.out)[at] = (bf16)v;
          }
        }
      }
    }
  }

  if constexpr (E == LSE) {
    // Tokens lie along lanes, the vocabulary along registers: a token's
    // maximum and sum need one exchange between the lane halves and one
    // between the two waves that share its column.
    __shared__ float2 half[2][kTile];
    float bias[2][16];
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const long long v = m0 + i * 32 + acc_row(r, lane);
        float b = 0.f;
        if (p.bias && v < M)
          b = SA == F32
              ? static_cast<const float*>(p.bias)[g * p.bias_group + v]
              : (float)static_cast<const bf16*>(p.bias)[g * p.bias_group + v];
        bias[i][r] = b;
      }
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const long long n = n0 + j * 32 + (lane & 31);
      const long long tgt = n < N ? p.target[g * N + n] : -1;
      float mx = -INFINITY;
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const long long v = m0 + i * 32 + acc_row(r, lane);
          float z = acc[i][j][r] + bias[i][r];
          if (v >= M) z = -INFINITY;
          else if (v == tgt) p.picked[g * N + n] = z;
          acc[i][j][r] = z;
          mx = fmaxf(mx, z);
        }
      mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
      const float ref = mx == -INFINITY ? 0.f : mx;
      float sum = 0.f;
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r)
          sum += __builtin_amdgcn_exp2f((acc[i][j][r] - ref) * kLog2e);
      sum += __shfl_xor(sum, 32, 64);
      if (lane < 32) half[wave >> 1][wn + j * 32 + lane] = make_float2(mx, sum);
    }
    __syncthreads();
    if (threadIdx.x < kTile) {
      const long long n = (long long)tn * kTile + threadIdx.x;
      if (n < N) {
        const float2 x = half[0][threadIdx.x], y = half[1][threadIdx.x];
        const float mx = fmaxf(x.x, y.x);
        const float ref = mx == -INFINITY ? 0.f : mx;
        p.part[(g * p.tiles_m + tm) * N + n] = make_float2(
            mx, x.y * __builtin_amdgcn_exp2f((x.x - ref) * kLog2e)
                    + y.y * __builtin_amdgcn_exp2f((y.x - ref) * kLog2e));
      }
    }
  }

  if constexpr (E == GRAD) {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const long long n = n0 + j * 32 + (lane & 31);
      long long tgt = p.ignore;
      float lse = 0.f, gr = 0.f;
      if (n < N) {
        tgt = p.target[g * N + n];
        lse = p.lse[g * N + n];
        gr = p.grad[g * p.grad_g + n * p.grad_n];
        if (p.count) gr /= p.count[g];
      }
      const bool live = n < N && tgt != p.ignore;
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const long long v = m0 + i * 32 + acc_row(r, lane);
          float d = 0.f;
          if (live && v < M) {
            float z = acc[i][j][r];
            if (p.bias)
              z += SA == F32
                  ? static_cast<const float*>(p.bias)[g * p.bias_group + v]
                  : (float)static_cast<const bf16*>(
                        p.bias)[g * p.bias_group + v];
            d = __builtin_amdgcn_exp2f((z - lse) * kLog2e);
            if (p.v0 + v == tgt) d -= 1.f;
            d *= gr;
          }
          // whole tiles are written: readers need no bounds
          const long long at = g * p.out_group + v * p.out_ld + n;
          if (SA == F32)
            static_cast<float*>(p.out)[at] = d;
          else
            static_cast<bf16*>(p.out)[at] = (bf16)d;
        }
    }
  }
}

template <typename T>
__global__ __launch_bounds__(kThreads)
void join_kernel(const float* __restrict__ partial, int splits,
                 long long slab, long long m, long long n, T* out,
                 long long out_ld, long long out_group, const T* bias,
                 long long bias_group) {
  const long long step = (long long)gridDim.x * kThreads;
  for (long long i = (long long)blockIdx.x * kThreads + threadIdx.x; i < slab;
       i += step) {
    float s = 0.f;
    for (int k = 0; k < splits; ++k) s += partial[k * slab + i];
    const long long c = i % n, row = i / n, g = row / m, r = row - g * m;
    if (bias) s += to_f(bias[g * bias_group + c]);
    out[g * out_group + r * out_ld + c] = from_f<T>(s);
  }
}

// Merges the vocabulary tiles' (max, sum) of 32 tokens per block, 8 threads a
// token, and leaves the block's loss sum and count in 64 bits.
__global__ __launch_bounds__(kThreads)
void lse_kernel(const float2* __restrict__ part,
                const float* __restrict__ picked,
                const long long* __restrict__ target, long long ignore,
                long long vocab, int tiles, long long rows,
                float* __restrict__ lse, float* __restrict__ row_loss,
                double2* __restrict__ sums) {
  __shared__ float2 seg[8][32];
  const int tl = threadIdx.x & 31, sl = threadIdx.x >> 5;
  const long long g = blockIdx.y;
  for (long long blk = blockIdx.x; blk * 32 < rows; blk += gridDim.x) {
    const long long n = blk * 32 + tl;
    float mx = -INFINITY, sum = 0.f;
    if (n < rows) {
      const float2* q = part + g * tiles * rows + n;
      for (int t = sl; t < tiles; t += 8) {
        const float2 v = q[(long long)t * rows];
        const float m = fmaxf(mx, v.x);
        const float ref = m == -INFINITY ? 0.f : m;
        sum = sum * __builtin_amdgcn_exp2f((mx - ref) * kLog2e)
            + v.y * __builtin_amdgcn_exp2f((v.x - ref) * kLog2e);
        mx = m;
      }
    }
    seg[sl][tl] = make_float2(mx, sum);
    __syncthreads();
    if (sl == 0) {
      double loss = 0.0, cnt = 0.0;
      if (n < rows) {
#pragma unroll
        for (int t = 1; t < 8; ++t) {
          const float2 v = seg[t][tl];
          const float m = fmaxf(mx, v.x);
          const float ref = m == -INFINITY ? 0.f : m;
          sum = sum * __builtin_amdgcn_exp2f((mx - ref) * kLog2e)
              + v.y * __builtin_amdgcn_exp2f((v.x - ref) * kLog2e);
          mx = m;
        }
        const long long tgt = target[g * rows + n];
        float l = mx + logf(sum);
        float row = 0.f;
        if (tgt != ignore) {
          if (tgt < 0 || tgt >= vocab) l = NAN;   // no such word
          row = l - ((tgt < 0 || tgt >= vocab) ? 0.f : picked[g * rows + n]);
          loss = row;
          cnt = 1.0;
        }
        lse[g * rows + n] = l;
        row_loss[g * rows + n] = row;
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        loss += __shfl_xor(loss, o, 32);
        cnt += __shfl_xor(cnt, o, 32);
      }
      if (tl == 0 && sums)
        sums[g * ((rows + 31) / 32) + blk] = make_double2(loss, cnt);
    }
    __syncthreads();
  }
}

__global__ __launch_bounds__(kThreads)
void loss_sum_kernel(const double2* __restrict__ sums, long long blocks,
                     float* __restrict__ loss, float* __restrict__ count,
                     int mean) {
  __shared__ double2 red[4];
  const long long g = blockIdx.x;
  double s = 0.0, c = 0.0;
  for (long long i = threadIdx.x; i < blocks; i += kThreads) {
    const double2 v = sums[g * blocks + i];
    s += v.x;
    c += v.y;
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    s += __shfl_xor(s, o, 64);
    c += __shfl_xor(c, o, 64);
  }
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = make_double2(s, c);
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < 4; ++w) { s += red[w].x; c += red[w].y; }
    loss[g] = (float)(mean ? s / c : s);          // 0 / 0: no counted row
    count[g] = (float)c;
  }
}

// A wave sums a row of the logits' gradient.
template <typename T>
__global__ __launch_bounds__(kThreads)
void rowsum_kernel(const T* __restrict__ pt, long long ld, long long group,
                   long long rows, long long cols, T* out,
                   long long out_group) {
  constexpr int V = Vec16<T>::n;
  const int lane = threadIdx.x & 63;
  const long long g = blockIdx.y;
  for (long long r = (long long)blockIdx.x * 4 + (threadIdx.x >> 6); r < rows;
       r += (long long)gridDim.x * 4) {
    const T* p = pt + g * group + r * ld;
    float s = 0.f;
    for (long long c = lane * V; c < cols; c += 64 * V) {
      float v[V];
      load_n<V>(p + c, v);
#pragma unroll
      for (int j = 0; j < V; ++j) s += v[j];
    }
    s = lanes_sum<64>(s);
    if (lane == 0) out[g * out_group + r] = from_f<T>(s);
  }
}

bool aligned(const void* p, long long n) {
  return reinterpret_cast<uintptr_t>(p) % (uintptr_t)n == 0;
}

// 16-byte loads (8 for 8-bit storage) are possible: aligned rows, and the
// contiguous axis ends on a whole access.
bool vector_ok(const Op& o, Src s) {
  const long long per = s == F32 ? 4 : 8, bytes = s == ACT8 ? 8 : 16;
  return o.ext % per == 0 && o.ld % per == 0 && o.group % per == 0
      && aligned(o.p, bytes);
}

Op make_op(const Mat& m, bool kmajor, long long rows, long long k) {
  Op o;
  o.p = m.p;
  o.ld = m.ld;
  o.group = m.group;
  o.rows = rows;
  o.ext = m.padded ? m.ld : kmajor ? rows : k;
  o.e = m.e;
  o.e_ld = m.e_ld;
  o.e_group = m.e_group;
  return o;
}

template <Src SA, bool KMA, Src SB, bool KMB, Epi E>
void launch(Params& p, long long groups, hipStream_t s) {
  const dim3 grid((unsigned)(p.tiles_m * p.tiles_n), (unsigned)p.splits,
                  (unsigned)groups);
  if (vector_ok(p.a, SA) && vector_ok(p.b, SB))
    gemm_kernel<SA, KMA, SB, KMB, true, E><<<grid, kThreads, 0, s>>>(p);
  else
    gemm_kernel<SA, KMA, SB, KMB, false, E><<<grid, kThreads, 0, s>>>(p);
}

unsigned grid_of(long long blocks) {
  return (unsigned)std::min<long long>(std::max<long long>(blocks, 1),
                                       1 << 20);
}

}  // namespace

// Parts to cut the contraction into: enough blocks for two per compute unit,
// each part at least 256 deep so that its sum is worth its trip to memory.
int gemm_splits(long long groups, long long m, long long n, long long k) {
  const long long tiles = ceil_div(m, kTile) * ceil_div(n, kTile) * groups;
  const long long want = ceil_div(512, std::max<long long>(tiles, 1));
  return (int)std::max<long long>(1, std::min(want, k / 256));
}

void gemm(const Gemm& g, hipStream_t s) {
  Params p = {};
  p.a = make_op(g.a, g.a_kmajor, g.m, g.k);
  p.b = make_op(g.b, g.b_kmajor, g.n, g.k);
  p.k = g.k;
  p.tiles_m = (int)ceil_div(g.m, kTile);
  p.tiles_n = (int)ceil_div(g.n, kTile);
  p.splits = g.partial ? g.splits : 1;
  p.out = g.out;
  p.out_ld = g.out_ld;
  p.out_group = g.out_group;
  p.out_f32 = g.tout == kF32;
  p.accumulate = g.accumulate;
  p.bias = g.bias;
  p.bias_group = g.bias_group;
  p.partial = g.partial;
  const bool f = g.ta == kF32;
  if (g.b.e) {                                     // dY' X8
    if (f) launch<F32, true, ACT8, true, STORE>(p, g.groups, s);
    else launch<BF16, true, ACT8, true, STORE>(p, g.groups, s);
  } else if (!g.a_kmajor && !g.b_kmajor) {         // X W'
    if (f) launch<F32, false, F32, false, STORE>(p, g.groups, s);
    else launch<BF16, false, BF16, false, STORE>(p, g.groups, s);
  } else if (!g.a_kmajor) {                        // dY W
    if (f) launch<F32, false, F32, true, STORE>(p, g.groups, s);
    else launch<BF16, false, BF16, true, STORE>(p, g.groups, s);
  } else {                                         // P' W, P stored by word
    if (f) launch<F32, true, F32, true, STORE>(p, g.groups, s);
    else launch<BF16, true, BF16, true, STORE>(p, g.groups, s);
  }
}

void join_partials(const float* partial, int splits, long long groups,
                   long long m, long long n, void* out, long long out_ld,
                   long long out_group, const void* bias,
                   long long bias_group, DType tout, hipStream_t s) {
  const long long slab = groups * m * n;
  const unsigned grid = grid_of(ceil_div(slab, kThreads));
  if (tout == kF32)
    join_kernel<float><<<grid, kThreads, 0, s>>>(
        partial, splits, slab, m, n, static_cast<float*>(out), out_ld,
        out_group, static_cast<const float*>(bias), bias_group);
  else
    join_kernel<bf16><<<grid, kThreads, 0, s>>>(
        partial, splits, slab, m, n, static_cast<bf16*>(out), out_ld,
        out_group, static_cast<const bf16*>(bias), bias_group);
}

long long loss_tiles(long long vocab) { return ceil_div(vocab, kTile); }
long long loss_sum_blocks(long long rows) { return ceil_div(rows, 32); }

namespace {
Params loss_params(const Loss& l, long long v0, long long nv) {
  Params p = {};
  const long long size = l.t == kF32 ? 4 : 2;
  Mat w = l.w;
  w.p = static_cast<const char*>(w.p) + v0 * w.ld * size;
  p.a = make_op(w, false, nv, l.dim);
  p.b = make_op(l.x, false, l.rows, l.dim);
  p.k = l.dim;
  p.tiles_m = (int)ceil_div(nv, kTile);
  p.tiles_n = (int)ceil_div(l.rows, kTile);
  p.splits = 1;
  p.bias = l.bias ? static_cast<const char*>(l.bias) + v0 * size : nullptr;
  p.bias_group = l.bias_group;
  p.target = l.target;
  p.ignore = l.ignore;
  p.v0 = v0;
  return p;
}
}  // namespace

void loss_forward(const Loss& l, void* part, float* picked, float* lse,
                  float* row_loss, void* block_sums, float* loss,
                  float* count, bool mean, hipStream_t s) {
  Params p = loss_params(l, 0, l.vocab);
  p.part = static_cast<float2*>(part);
  p.picked = picked;
  if (l.t == kF32) launch<F32, false, F32, false, LSE>(p, l.groups, s);
  else launch<BF16, false, BF16, false, LSE>(p, l.groups, s);
  const long long blocks = loss_sum_blocks(l.rows);
  lse_kernel<<<dim3(grid_of(blocks), (unsigned)l.groups), kThreads, 0, s>>>(
      p.part, picked, l.target, l.ignore, l.vocab, p.tiles_m, l.rows, lse,
      row_loss, static_cast<double2*>(block_sums));
  if (loss)
    loss_sum_kernel<<<dim3((unsigned)l.groups), kThreads, 0, s>>>(
        static_cast<const double2*>(block_sums), blocks, loss, count, mean);
}

void loss_logit_grad(const Loss& l, long long v0, long long nv,
                     const float* lse, const float* grad, long long grad_g,
                     long long grad_n, const float* count, void* pt,
                     long long pt_ld, long long pt_group, hipStream_t s) {
  Params p = loss_params(l, v0, nv);
  p.lse = lse;
  p.grad = grad;
  p.grad_g = grad_g;
  p.grad_n = grad_n;
  p.count = count;
  p.out = pt;
  p.out_ld = pt_ld;
  p.out_group = pt_group;
  if (l.t == kF32) launch<F32, false, F32, false, GRAD>(p, l.groups, s);
  else launch<BF16, false, BF16, false, GRAD>(p, l.groups, s);
}

void rowsum(const void* pt, long long ld, long long group, long long groups,
            long long rows, long long cols, void* out, long long out_group,
            DType t, hipStream_t s) {
  const dim3 grid(grid_of(ceil_div(rows, 4)), (unsigned)groups);
  if (t == kF32)
    rowsum_kernel<float><<<grid, kThreads, 0, s>>>(
        static_cast<const float*>(pt), ld, group, rows, cols,
        static_cast<float*>(out), out_group);
  else
    rowsum_kernel<bf16><<<grid, kThreads, 0, s>>>(
        static_cast<const bf16*>(pt), ld, group, rows, cols,
        static_cast<bf16*>(out), out_group);
}

}  // namespace token_ops
