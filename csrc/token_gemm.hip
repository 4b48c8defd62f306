// Matrix products on the matrix cores for the linear layers of token models,
// with the epilogues of a large-vocabulary loss.
//
// One tile loop serves every product; operands differ in
//   * type: bf16 as it is; fp32 cut into three bf16 parts; 8-bit activations
//     (act8.hip), whose stored values are exact in bf16;
//   * order: contraction along the rows ([m][k]) or across them ([k][m]).
//
// fp32: x = hi + mid + lo, each the nearest bf16 to what is left, is exact:
// |mid| <= 2^-8 and |lo| <= 2^-17 of a power of two not above |x|.  The six
// products hi*hi, hi*mid, mid*hi, hi*lo, mid*mid, lo*hi leave out mid*lo,
// lo*mid and lo*lo, at most 2^-24 of |a||b| (half a step of fp32) and of
// either sign.  (Parts cut off instead of rounded are twice and four times as
// large and have the operand's sign: up to 2^-21 left out, always towards
// zero.)  Six bf16 products per multiplication have 2.6 times the rate of the
// fp32 matrix instruction.
// A value that is not finite makes its results NaN (inf - inf in the parts).
//
// A block owns 256 x 256, 128 x 128 or 64 x 64 of the output (tiling() below
// chooses) in v_mfma_f32_32x32x16_bf16 tiles.  LDS holds two steps: one is
// multiplied while the next is converted and written, and loads beyond it are
// on their way in registers.
//   [m][k] tiles lie in LDS as [rows][BK] with 16-byte columns swizzled by the
//   row: the 16-byte fragment reads touch every bank once.
//   [k][m] tiles lie as [BK][rows] and are read by ds_read_b64_tr_b16, which
//   hands each lane 4 values down a column; 32-byte columns swizzled by k.
// Sums are 32-bit in the accumulators.
//
// Bound by the matrix units: 54 to 68 percent busy in the long bf16 products
// (the library's have 63 to 75), 52 to 59 in fp32 ones of a few hundred deep
// and many blocks, 25 to 45 where a block's few steps do not cover its start
// and its output.  Logits 8192 x 50021 x 2048 bf16 in 1470 to 1520 us, 1100 to
// 1140 TFLOP/s; fp32 logits 16 x 500 x 10000 x 300 in 290 to 316 us, 152 to
// 166 TFLOP/s, and products with their gradient 118 to 130: about what the
// library's fp32 product reaches at its best sizes (154).

#include "token_ops.h"
#include "token_device.h"

#include <algorithm>
#include <type_traits>

namespace token_ops {
namespace {

constexpr int kThreads = 256;          // of the small kernels below

enum Src { F32, BF16, ACT8 };
enum Epi { STORE, LSE, GRAD };
enum Size { TINY, SMALL, LARGE };

template <Src S> struct SrcOf;
template <> struct SrcOf<F32> { using T = float; static constexpr int P = 3; };
template <> struct SrcOf<BF16> { using T = bf16; static constexpr int P = 1; };
template <> struct SrcOf<ACT8> {
  using T = int8_t;
  static constexpr int P = 1;
};

// Waves of a block along m and n, each wave's 32 x 32 tiles, and the depth of
// a step for one-part and for three-part operands.
template <int WM_, int WN_, int MF_, int NF_, int BK1_, int BK3_>
struct Shape {
  static constexpr int WM = WM_, WN = WN_, MF = MF_, NF = NF_;
  static constexpr int BK1 = BK1_, BK3 = BK3_;
  static constexpr int BM = WM * MF * 32, BN = WN * NF * 32;
  static constexpr int THREADS = WM * WN * 64;
};
using Tiny = Shape<2, 2, 1, 1, 64, 32>;    // 64 x 64, 4 waves
using Small = Shape<2, 2, 2, 2, 64, 16>;   // 128 x 128, 4 waves
using Large = Shape<2, 4, 4, 2, 64, 16>;   // 256 x 256, 8 waves

// What a kernel knows of an operand: `rows` of the output it feeds (m or n),
// and how far the contiguous axis may be read.
struct Op {
  const void* p;
  long long ld, group;
  int rows, ext;
  const uint8_t* e;
  long long e_ld, e_group;
};

struct Params {
  Op a, b;
  int k;
  int tiles_m, tiles_n, splits;
  // STORE
  void* out;
  long long out_ld, out_group;
  int accumulate;
  const void* bias;
  long long bias_group;
  float* partial;
  // LSE, GRAD: m runs over the vocabulary, n over the tokens
  const long long* target;
  long long ignore, v0;
  float2* part;
  float* picked;
  const float2* lse;      // a row's maximum, and its sum's logarithm from there
  const float* ratio;     // [groups][n], null: all ones
  float* rowsum;          // [groups][tiles_n * WN][m], may be null
  Scale scale;            // of what STORE writes
};

// The nearest bf16 to two floats, packed; a and b keep what is left.
__device__ __forceinline__ uint32_t take_bf16(float na, float nb, float& a,
                                              float& b) {
  const bf16x2 t = {(bf16)na, (bf16)nb};
  const uint32_t u = __builtin_bit_cast(uint32_t, t);
  a -= __uint_as_float(u << 16);
  b -= __uint_as_float(u & 0xffff0000u);
  return u;
}

// Three bf16 parts of 8 floats, packed in pairs.
__device__ __forceinline__ void split3(const float (&x)[8], u32x4 (&o)[3]) {
  // bf16's largest value: what would round beyond it leaves more to mid
  constexpr float kMost = 0x1.fep127f;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    float a = x[2 * j], b = x[2 * j + 1];
    o[0][j] = take_bf16(__builtin_amdgcn_fmed3f(a, -kMost, kMost),
                        __builtin_amdgcn_fmed3f(b, -kMost, kMost), a, b);
    o[1][j] = take_bf16(a, b, a, b);
    o[2][j] = take_bf16(a, b, a, b);
  }
}

// Wide accesses at an element's alignment: rows of any length and stride are
// read 16 bytes at a time.
typedef f32x4 f32x4_u __attribute__((aligned(4)));
typedef u32x4 u32x4_u __attribute__((aligned(2)));
typedef u32x2 u32x2_u __attribute__((aligned(1)));
typedef bf16x8 bf16x8_u __attribute__((aligned(2)));

template <typename T>
using Global = const __attribute__((address_space(1))) T*;

// A pointer that is the same for all threads, held in scalar registers: left
// to itself the compiler adds each thread's offset to it once and keeps the
// sums, two registers a chunk, and spills (8-bit weight gradient 32768 x 4096
// x 1024: 11 % slower so; other products 1 to 4 %).
template <typename T>
__device__ __forceinline__ Global<T> scalar(Global<T> p) {
  const uint64_t u = reinterpret_cast<uint64_t>(p);
  const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)u);
  const uint32_t hi = __builtin_amdgcn_readfirstlane((uint32_t)(u >> 32));
  return reinterpret_cast<Global<T>>((uint64_t)hi << 32 | lo);
}

template <Src S> struct Raw { u32x4 v; };
template <> struct Raw<F32> { f32x4 x, y; };
template <> struct Raw<ACT8> { u32x2 v; uint32_t e; };

// Moves one operand's ROWS x BK tile: global -> registers -> LDS, in chunks
// of 8 values along the contiguous axis.
template <Src S, bool KM, int ROWS, int THREADS, int BK, int SETS_>
struct Loader {
  using T = typename SrcOf<S>::T;
  static constexpr int P = SrcOf<S>::P;
  static constexpr int N = ROWS * BK / 8 / THREADS;     // chunks a thread
  static constexpr int PLANE = ROWS * BK;               // bf16 values
  static_assert(N >= 1 && N * 8 * THREADS == ROWS * BK);
  Global<char> base;     // the next step's tile, the same for all threads
  Global<uint8_t> ebase;
  uint32_t off[N], eoff[N];                // bytes from there to a chunk
  long long ld, e_ld;
  int ext, left[N];      // [k][m]: end of a row, values from a chunk to it
  int kend, krows;       // end of this block's and of the whole contraction
  static constexpr int SETS = SETS_;      // steps on their way
  Raw<S> raws[SETS][N];

  __device__ __forceinline__ void init(const Op& o, long long g, int tile,
                                       int k0, int kend_, int krows_) {
    ld = o.ld;
    e_ld = o.e_ld;
    ext = o.ext;
    kend = kend_;
    krows = krows_;
    const int row0 = tile * ROWS;
    base = (Global<char>)o.p
        + (g * o.group + (KM ? k0 * ld + row0 : row0 * ld + k0)) * sizeof(T);
    if constexpr (S == ACT8)
      ebase = (Global<uint8_t>)o.e + g * o.e_group + k0 * e_ld + (row0 >> 7);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int id = i * THREADS + threadIdx.x;
      // Rows (or columns) beyond the operand feed outputs that nobody
      // stores: read its last ones for them.
      if constexpr (KM) {
        const int k = id / (ROWS / 8);
        int c = id % (ROWS / 8) * 8;
        const int last = ((ext - 1) & ~7) - row0;
        if (c > last) c = last;
        left[i] = ext - row0 - c;
        off[i] = (uint32_t)((k * ld + c) * sizeof(T));
        if constexpr (S == ACT8)
          eoff[i] = (uint32_t)(k * e_ld + (c >> 7));
      } else {
        int r = id / (BK / 8);
        if (r >= o.rows - row0) r = o.rows - row0 - 1;
        off[i] = (uint32_t)((r * ld + id % (BK / 8) * 8) * sizeof(T));
      }
    }
  }

  __device__ __forceinline__ Global<T> at(int i) const {
    return reinterpret_cast<Global<T>>(base + off[i]);
  }
  __device__ __forceinline__ void advance() {
    base += (KM ? BK * ld : (long long)BK) * (long long)sizeof(T);
    base = scalar(base);
    if constexpr (S == ACT8) ebase = scalar(ebase + BK * e_ld);
  }

  // Whether the step from k0 can be read as it lies.  A [k][m] row's last
  // chunk may run up to 7 values into the rows behind it, which have to be
  // there.
  __device__ __forceinline__ bool whole(int k0) const {
    return k0 + BK <= kend
        && (!KM || (ext & 7) == 0 || (krows - k0 - BK) * ld >= 8);
  }

  template <int SET> __device__ __forceinline__ void load_whole() {
    Raw<S>(&raw)[N] = raws[SET];
#pragma unroll
    for (int i = 0; i < N; ++i) {
      // 32 bits here, widened by the load itself
      asm("" : "+v"(off[i]));
      if constexpr (S == F32) {
        raw[i].x = *reinterpret_cast<Global<f32x4_u>>(at(i));
        raw[i].y = *reinterpret_cast<Global<f32x4_u>>(at(i) + 4);
      } else if constexpr (S == BF16) {
        raw[i].v = *reinterpret_cast<Global<u32x4_u>>(at(i));
      } else {
        raw[i].v = *reinterpret_cast<Global<u32x2_u>>(at(i));
        raw[i].e = ebase[eoff[i]];
      }
    }
    advance();
  }

  template <int SET> __device__ __forceinline__ void load(int k0) {
    if (whole(k0)) load_whole<SET>(); else tail(k0, raws[SET]);
  }

  // The last step: each value is checked, and zero beyond the contraction.
  __device__ __forceinline__ void tail(int k0, Raw<S> (&raw)[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int id = i * THREADS + threadIdx.x;
      int valid;
      if constexpr (KM) {
        const bool in = k0 + id / (ROWS / 8) < kend;
        valid = !in ? 0 : left[i] < 8 ? left[i] : 8;
      } else {
        valid = kend - (k0 + id % (BK / 8) * 8);
      }
      if constexpr (S == F32) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          raw[i].x[j] = j < valid ? at(i)[j] : 0.f;
          raw[i].y[j] = 4 + j < valid ? at(i)[4 + j] : 0.f;
        }
      } else if constexpr (S == BF16) {
        const Global<uint16_t> h = reinterpret_cast<Global<uint16_t>>(at(i));
        raw[i].v = u32x4{0, 0, 0, 0};
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (j < valid) raw[i].v[j >> 1] |= (uint32_t)h[j] << (16 * (j & 1));
      } else {
        const Global<uint8_t> h = reinterpret_cast<Global<uint8_t>>(at(i));
        raw[i].v = u32x2{0, 0};
        raw[i].e = valid > 0 ? ebase[eoff[i]] : 0;
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (j < valid) raw[i].v[j >> 2] |= (uint32_t)h[j] << (8 * (j & 3));
      }
    }
    advance();
  }

  template <int SET>
  __device__ __forceinline__ void store(bf16* lds) const {
    const Raw<S>(&raw)[N] = raws[SET];
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int id = i * THREADS + threadIdx.x;
      int at;
      if constexpr (KM) {
        const int k = id / (ROWS / 8), c = id % (ROWS / 8);
        at = k * ROWS + (((c >> 1) ^ swap(k)) << 4) + (c & 1) * 8;
      } else {
        const int r = id / (BK / 8), c = id % (BK / 8);
        at = r * BK + ((c ^ swizzle(r)) << 3);
      }
      u32x4 o[3];
      if constexpr (S == F32) {
        float v[8];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          v[j] = raw[i].x[j];
          v[4 + j] = raw[i].y[j];
        }
        split3(v, o);
      } else if constexpr (S == BF16) {
        o[0] = raw[i].v;
      } else {
        // Bytes convert unsigned; (q + 128) - 128 and its product with a
        // power of two are exact.  (One fma with -128 * unit would overflow
        // for blocks that reach 2^127.)
        const float unit = __uint_as_float(raw[i].e << 23);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint32_t w = raw[i].v[h] ^ 0x80808080u;
          float v[4];
#pragma unroll
          for (int t = 0; t < 4; ++t)
            v[t] = ((float)((w >> (8 * t)) & 0xffu) - 128.f) * unit;
          o[0][2 * h] = __builtin_amdgcn_perm(
              __float_as_uint(v[1]), __float_as_uint(v[0]), 0x07060302u);
          o[0][2 * h + 1] = __builtin_amdgcn_perm(
              __float_as_uint(v[3]), __float_as_uint(v[2]), 0x07060302u);
        }
      }
#pragma unroll
      for (int q = 0; q < P; ++q)
        *reinterpret_cast<u32x4*>(lds + q * PLANE + at) = o[q];
    }
  }

  // 16-byte columns of an [m][BK] row are swapped about by the row so that 16
  // neighbouring rows' reads of one column touch each of the 64 banks once.
  static __device__ __forceinline__ int swizzle(int r) {
    constexpr int C = BK / 8;                 // columns; 16 / C rows a bank row
    return r / (16 / C) % C;
  }

  // 32-byte columns of a [BK][m] row likewise by k, so that the 4 rows and 2
  // columns of a transposing read touch each bank once; k + 4 goes as k does.
  static __device__ __forceinline__ int swap(int k) {
    return ROWS >= 128 ? 2 * (k & 3) : 2 * ((k >> 1) & 1);
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
      const bf16* q = lds + k * ROWS + ((c ^ swap(k)) << 4)
          + (i & 3) * 4;
      union { s4 h[2]; bf16x8 v; } u;
      typedef __attribute__((address_space(3))) s4* lds_s4;
      u.h[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4)(q));
      u.h[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
          (lds_s4)(q + 4 * ROWS));
      return u.v;
    } else {
      const int r = base + (lane & 31);
      const int c = ks * 2 + (lane >> 5);
      return *reinterpret_cast<const bf16x8*>(
          lds + r * BK + ((c ^ swizzle(r)) << 3));
    }
  }
};

// Row of accumulator element r, for the 32 x 32 tile's lane half.
__device__ __forceinline__ int acc_row(int r, int lane) {
  return (r & 3) + 8 * (r >> 2) + 4 * (lane >> 5);
}

// Of 2 * LEN values, lanes without bit `o` keep the sums of the first half,
// lanes with it those of the second.
template <int LEN, int N>
__device__ __forceinline__ void fold(float (&sum)[N], int o, int lane,
                                     int& lo) {
  const bool up = lane & o;
#pragma unroll
  for (int i = 0; i < LEN; ++i) {
    const float mine = up ? sum[LEN + i] : sum[i];
    const float other = up ? sum[i] : sum[LEN + i];
    sum[i] = mine + __shfl_xor(other, o, 64);
  }
  if (up) lo += LEN;
}

// LDS written by other lanes of the wave before it can be read behind it.
__device__ __forceinline__ void wave_fence() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

constexpr float kLog2e = 1.4426950408889634f;

template <Src S>
__device__ __forceinline__ float bias_at(const void* p, long long i) {
  return S == F32 ? static_cast<const float*>(p)[i]
                  : (float)static_cast<const bf16*>(p)[i];
}

template <Src SA, bool KMA, Src SB, bool KMB, typename H, Epi E>
// Small fp32 blocks are held to 168 registers so that three share a compute
// unit: 7 % less time for the two gradient products of 16 x 500 x 5000 x 300.
__global__ __launch_bounds__(H::THREADS,
                             SrcOf<SA>::P == 3 && H::MF == 2 ? 3 : 1)
void gemm_kernel(Params p) {
  constexpr int PA = SrcOf<SA>::P, PB = SrcOf<SB>::P;
  constexpr int MF = H::MF, NF = H::NF;
  constexpr int BK = (PA == 3 || PB == 3) ? H::BK3 : H::BK1;
  // a step of fp32 or of a tiny tile is short against memory's latency: two
  // are on their way
  constexpr int SETS = BK == H::BK3 || H::MF == 1 ? 2 : 1;
  using LA = Loader<SA, KMA, H::BM, H::THREADS, BK, SETS>;
  using LB = Loader<SB, KMB, H::BN, H::THREADS, BK, SETS>;
  __shared__ __attribute__((aligned(16))) bf16 sa[2][PA * LA::PLANE];
  __shared__ __attribute__((aligned(16))) bf16 sb[2][PB * LB::PLANE];

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
  const int steps = (p.k + BK - 1) / BK;
  const int s0 = (int)((long long)steps * split / p.splits);
  const int s1 = (int)((long long)steps * (split + 1) / p.splits);
  const int kend = (long long)s1 * BK < p.k ? s1 * BK : p.k;

  LA la;
  LB lb;
  la.init(p.a, g, tm, s0 * BK, kend, p.k);
  lb.init(p.b, g, tn, s0 * BK, kend, p.k);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int wm = wave / H::WN * (MF * 32), wn = wave % H::WN * (NF * 32);

  f32x16 acc[MF][NF];
#pragma unroll
  for (int i = 0; i < MF; ++i)
#pragma unroll
    for (int j = 0; j < NF; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.f;

  // Units of a step: one 16-deep slice of one row of the wave's tiles.
  constexpr int UNITS = BK / 16 * MF;
  bf16x8 fbs[2][NF][PB];                 // of even and odd slices
  auto read_b = [&](const bf16* tb, int ks) {
#pragma unroll
    for (int j = 0; j < NF; ++j)
#pragma unroll
      for (int q = 0; q < PB; ++q)
        fbs[ks & 1][j][q] = LB::frag(tb + q * LB::PLANE, wn + j * 32, ks);
  };
  auto read_a = [&](const bf16* ta, int u, bf16x8 (&fa)[PA]) {
#pragma unroll
    for (int q = 0; q < PA; ++q)
      fa[q] = LA::frag(ta + q * LA::PLANE, wm + u % MF * 32, u / MF);
  };
  // bf16 outputs are computed transposed, with m along the lanes: a lane's
  // values lie along a row and go to LDS, and from there to memory, 16 bytes
  // at a time.
  constexpr bool ACROSS = E == STORE && SA == BF16;
  auto products = [&](int u, const bf16x8 (&fa)[PA]) {
    const int i = u % MF;
    const bf16x8(&fb)[NF][PB] = fbs[u / MF & 1];
#pragma unroll
    for (int qa = 0; qa < PA; ++qa)
#pragma unroll
      for (int qb = 0; qb < PB; ++qb) {
        if (qa + qb > 2) continue;
#pragma unroll
        for (int j = 0; j < NF; ++j)
          acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(
              ACROSS ? fb[j][qb] : fa[qa], ACROSS ? fa[qa] : fb[j][qb],
              acc[i][j], 0, 0, 0);
      }
  };
  auto multiply = [&](const bf16* ta, const bf16* tb) {
#pragma unroll
    for (int u = 0; u < UNITS; ++u) {
      if (u % MF == 0) read_b(tb, u / MF);
      bf16x8 fa[PA];
      read_a(ta, u, fa);
      products(u, fa);
    }
  };
  // Transposing reads, two to a fragment, are issued one unit ahead of their
  // products (bf16 P'W 8192 x 2048 x 12544 4 % faster, dY'X8 32768 x 4096 x
  // 1024 8 %); plain ones are better left to the compiler (logits 8192 x 50021
  // x 2048 10 % slower, and 1 % where whole slices are read ahead).
  constexpr bool AHEAD = KMA || KMB;
  constexpr int FIRST = MF;      // units that cover conversion and writing

  // Two tiles in LDS: one is multiplied while the next is converted and
  // written, and the one or two after it are on their way in registers.  One
  // barrier a step: behind it the tile to multiply is whole and the other
  // one free.
  auto fast_step = [&](auto cur, auto set) {
    __syncthreads();
    // The fragments come first: a read cannot pass the writes below.
    __builtin_amdgcn_sched_barrier(0);
    read_b(sb[cur()], 0);
    bf16x8 fa[FIRST][PA];
#pragma unroll
    for (int u = 0; u < FIRST; ++u) read_a(sa[cur()], u, fa[u]);
    bf16x8 ahead[2][PA];
    if (AHEAD && UNITS > FIRST) {
      read_b(sb[cur()], 1);
      read_a(sa[cur()], FIRST, ahead[FIRST & 1]);
    }
    __builtin_amdgcn_sched_barrier(0);
    la.template store<decltype(set)::value>(sa[cur() ^ 1]);
    lb.template store<decltype(set)::value>(sb[cur() ^ 1]);
#pragma unroll
    for (int u = 0; u < FIRST; ++u) products(u, fa[u]);
    // one product, then what the vector unit does in its shadow: its work
    // spread over the products (8-bit values need the most conversion)
    constexpr int SHADE = PA == 1 && SB == ACT8 ? 12 : 4;
#pragma unroll
    for (int q = 0; q < FIRST * NF * (PA * PB > 3 ? 6 : PA * PB); ++q) {
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
      __builtin_amdgcn_sched_group_barrier(0x002, SHADE, 0);
      __builtin_amdgcn_sched_group_barrier(0x200, 1, 0);
    }
    // Left to itself the compiler moves these loads behind the products.
    __builtin_amdgcn_sched_barrier(0);
    la.template load_whole<decltype(set)::value>();
    lb.template load_whole<decltype(set)::value>();
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int u = FIRST; u < UNITS; ++u) {
      if (AHEAD) {
        if (u + 1 < UNITS) {
          if ((u + 1) % MF == 0) read_b(sb[cur()], (u + 1) / MF);
          read_a(sa[cur()], u + 1, ahead[(u + 1) & 1]);
        }
        __builtin_amdgcn_sched_barrier(0);
        products(u, ahead[u & 1]);
        __builtin_amdgcn_sched_barrier(0);
      } else {
        if (u % MF == 0) read_b(sb[cur()], u / MF);
        read_a(sa[cur()], u, ahead[0]);
        products(u, ahead[0]);
      }
    }
  };
  auto checked_step = [&](int s, auto cur, auto set) {
    __syncthreads();
    if (s + 1 < s1) {
      la.template store<decltype(set)::value>(sa[cur() ^ 1]);
      lb.template store<decltype(set)::value>(sb[cur() ^ 1]);
    }
    if (s + 1 + SETS < s1) {
      la.template load<decltype(set)::value>((s + 1 + SETS) * BK);
      lb.template load<decltype(set)::value>((s + 1 + SETS) * BK);
    }
    multiply(sa[cur()], sb[cur()]);
  };
  using Zero = std::integral_constant<int, 0>;
  using One = std::integral_constant<int, 1>;
  // the register set of odd steps
  using Odd = std::integral_constant<int, SETS - 1>;

  int s = s0;
  // Every step before the last is whole unless an operand's rows are shorter
  // than a chunk; without a branch, conversion and loads go between the
  // matrix instructions.
  if (s0 + SETS + 3 < s1 && (!KMA || p.a.ld >= 8) && (!KMB || p.b.ld >= 8)) {
    la.template load_whole<0>();
    lb.template load_whole<0>();
    la.template store<0>(sa[0]);
    lb.template store<0>(sb[0]);
    la.template load_whole<Odd::value>();
    lb.template load_whole<Odd::value>();
    if (SETS == 2) {
      la.template load_whole<0>();
      lb.template load_whole<0>();
    }
    do {
      fast_step(Zero(), Odd());
      fast_step(One(), Zero());
      s += 2;
    } while (s + SETS + 3 < s1);
  } else {
    if (s0 < s1) {
      la.template load<0>(s0 * BK);
      lb.template load<0>(s0 * BK);
      la.template store<0>(sa[0]);
      lb.template store<0>(sb[0]);
    }
    if (s0 + 1 < s1) {
      la.template load<Odd::value>((s0 + 1) * BK);
      lb.template load<Odd::value>((s0 + 1) * BK);
    }
    if (SETS == 2 && s0 + 2 < s1) {
      la.template load<0>((s0 + 2) * BK);
      lb.template load<0>((s0 + 2) * BK);
    }
  }
  for (; s < s1; s += 2) {
    checked_step(s, Zero(), Odd());
    if (s + 1 < s1) checked_step(s + 1, One(), Zero());
  }

  const int m0 = tm * H::BM + wm, n0 = tn * H::BN + wn;
  const int M = p.a.rows, N = p.b.rows;

  if constexpr (ACROSS) {
    // Each wave passes 32 rows at a time through LDS of its own and writes
    // them in whole lines (32768 x 1024 x 4096: 426 us with a 2-byte store a
    // value, 287 so).
    constexpr int W = NF * 32, LD = W + 4;        // LD: rows on other banks
    constexpr int LANES = W / 8, HALF = H::WM * H::WN / 2;
    static_assert(HALF * 32 * LD * 4 <= 2 * LA::PLANE * 2
                  && HALF * 32 * LD * 4 <= 2 * LB::PLANE * 2);
    __syncthreads();                              // the tiles have been read
    float* stage = reinterpret_cast<float*>(wave < HALF ? sa[0] : sb[0])
        + wave % HALF * (32 * LD);
    const float scale = scale_of(p.scale, g);
    const bool finite = fabsf(scale) < INFINITY;
    const int c = lane % LANES * 8, n = n0 + c, left = N - n;
    float bias[8];
#pragma unroll
    for (int t = 0; t < 8; ++t)
      bias[t] = p.bias && !p.partial && t < left
          ? bias_at<BF16>(p.bias, g * p.bias_group + n + t) : 0.f;
#pragma unroll
    for (int i = 0; i < MF; ++i) {
#pragma unroll
      for (int j = 0; j < NF; ++j)
#pragma unroll
        for (int q = 0; q < 4; ++q)
          *reinterpret_cast<f32x4*>(
              stage + (lane & 31) * LD + j * 32 + acc_row(4 * q, lane)) =
              f32x4{acc[i][j][4 * q], acc[i][j][4 * q + 1],
                    acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]};
      wave_fence();
#pragma unroll
      for (int r0 = 0; r0 < 32; r0 += 64 / LANES) {
        const int row = r0 + lane / LANES, m = m0 + i * 32 + row;
        if (m >= M || left <= 0) continue;
        float v[8];
        load_n<8>(stage + row * LD + c, v);
#pragma unroll
        for (int t = 0; t < 8; ++t)
          v[t] = finite ? fmaf(v[t], scale, bias[t])
                        : scaled(v[t], scale) + bias[t];
        if (p.partial) {
          float* o = p.partial
              + (((long long)split * gridDim.z + g) * M + m) * N + n;
          if (left >= 8) {
#pragma unroll
            for (int t = 0; t < 8; t += 4) {
              f32x4 s = {v[t], v[t + 1], v[t + 2], v[t + 3]};
              f32x4_u* at = reinterpret_cast<f32x4_u*>(o + t);
              if (p.accumulate) s += *at;
              *at = s;
            }
          } else {
#pragma unroll
            for (int t = 0; t < 8; ++t)
              if (t < left) o[t] = p.accumulate ? o[t] + v[t] : v[t];
          }
        } else {
          bf16* o = static_cast<bf16*>(p.out) + g * p.out_group
              + (long long)m * p.out_ld + n;
          if (left >= 8) {
            bf16x8 s;
#pragma unroll
            for (int t = 0; t < 8; ++t) s[t] = (bf16)v[t];
            *reinterpret_cast<bf16x8_u*>(o) = s;
          } else {
#pragma unroll
            for (int t = 0; t < 8; ++t)
              if (t < left) o[t] = (bf16)v[t];
          }
        }
      }
      wave_fence();
    }
  } else if constexpr (E == STORE) {
    const float scale = scale_of(p.scale, g);
    const bool finite = fabsf(scale) < INFINITY;
#pragma unroll
    for (int j = 0; j < NF; ++j) {
      const int n = n0 + j * 32 + (lane & 31);
      if (n >= N) continue;
      float bias = 0.f;
      if (p.bias && !p.partial)
        bias = bias_at<F32>(p.bias, g * p.bias_group + n);
#pragma unroll
      for (int i = 0; i < MF; ++i) {
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int m = m0 + i * 32 + acc_row(r, lane);
          if (m >= M) continue;
          const float v = finite ? fmaf(acc[i][j][r], scale, bias)
                                 : scaled(acc[i][j][r], scale) + bias;
          if (p.partial) {
            float* o = p.partial
                + (((long long)split * gridDim.z + g) * M + m) * N + n;
            *o = p.accumulate ? *o + v : v;
          } else {
            static_cast<float*>(p.out)[g * p.out_group
                                       + (long long)m * p.out_ld + n] = v;
          }
        }
      }
    }
  }

  if constexpr (E != STORE) {
    // the tile's biases, -inf beyond the vocabulary
    float* sbias = reinterpret_cast<float*>(sa[0]);
    __syncthreads();
    for (int i = threadIdx.x; i < H::BM; i += H::THREADS) {
      const int v = tm * H::BM + i;
      sbias[i] = v >= M ? -INFINITY
          : p.bias ? bias_at<SA>(p.bias, g * p.bias_group + v) : 0.f;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < MF; ++i)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const f32x4 b = *reinterpret_cast<const f32x4*>(
            sbias + wm + i * 32 + acc_row(4 * q, lane));
#pragma unroll
        for (int j = 0; j < NF; ++j)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            // a row beyond the vocabulary holds another's product: replace
            const int m = m0 + i * 32 + acc_row(4 * q + r, lane);
            acc[i][j][4 * q + r] =
                m < M ? acc[i][j][4 * q + r] + b[r] : b[r];
          }
      }
  }

  if constexpr (E == LSE) {
    // Tokens lie along lanes, the vocabulary along registers: a token's
    // maximum and sum need one exchange between the lane halves and one
    // between the waves that share its column.
    float2* half = reinterpret_cast<float2*>(sb[0]);     // [WM][BN]
#pragma unroll
    for (int j = 0; j < NF; ++j) {
      const int n = n0 + j * 32 + (lane & 31);
      const long long tgt = n < N ? p.target[g * N + n] : -1;
      // the target's place in this wave's rows, or out of them
      const long long place = tgt - m0;
      const int row = place >= 0 && place < MF * 32 && tgt < M ? (int)place
                                                               : -1;
      float mx = -INFINITY;
#pragma unroll
      for (int i = 0; i < MF; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          mx = fmaxf(mx, acc[i][j][r]);
          if (i * 32 + acc_row(r, lane) == row)
            p.picked[g * N + n] = acc[i][j][r];
        }
      mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
      const float ref = mx == -INFINITY ? 0.f : mx;
      float sum = 0.f;
#pragma unroll
      for (int i = 0; i < MF; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r)
          sum += __builtin_amdgcn_exp2f((acc[i][j][r] - ref) * kLog2e);
      sum += __shfl_xor(sum, 32, 64);
      if (lane < 32)
        half[wave / H::WN * H::BN + wn + j * 32 + lane] = make_float2(mx, sum);
    }
    __syncthreads();
    for (int t = threadIdx.x; t < H::BN; t += H::THREADS) {
      const int n = tn * H::BN + t;
      if (n < N) {
        float mx = half[t].x;
#pragma unroll
        for (int w = 1; w < H::WM; ++w) mx = fmaxf(mx, half[w * H::BN + t].x);
        const float ref = mx == -INFINITY ? 0.f : mx;
        float sum = 0.f;
#pragma unroll
        for (int w = 0; w < H::WM; ++w) {
          const float2 x = half[w * H::BN + t];
          sum += x.y * __builtin_amdgcn_exp2f((x.x - ref) * kLog2e);
        }
        p.part[(g * p.tiles_m + tm) * N + n] = make_float2(mx, sum);
      }
    }
  }

  if constexpr (E == GRAD) {
    // sums over this wave's tokens, 32 lanes still apart
    float sum[MF * 16];
#pragma unroll
    for (int i = 0; i < MF * 16; ++i) sum[i] = 0.f;
#pragma unroll
    for (int j = 0; j < NF; ++j) {
      const int n = n0 + j * 32 + (lane & 31);
      long long tgt = p.ignore;
      float2 lse = {0.f, 0.f};
      float ratio = 1.f;
      if (n < N) {
        tgt = p.target[g * N + n];
        lse = p.lse[g * N + n];
        if (p.ratio) ratio = p.ratio[g * N + n];
      }
      const bool live = n < N && tgt != p.ignore;
      const float less = lse.y * -kLog2e;
      const long long place = tgt - p.v0 - m0;
      const int row = place >= 0 && place < MF * 32 ? (int)place : -1;
      // whole tiles are written: readers need no bounds
      const long long at = g * p.out_group
          + (long long)(m0 + 4 * (lane >> 5)) * p.out_ld + n;
#pragma unroll
      for (int i = 0; i < MF; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int mr = i * 32 + (r & 3) + 8 * (r >> 2);
          // beyond the vocabulary the logit is -inf: exp gives 0
          float d = __builtin_amdgcn_exp2f(
              fmaf(acc[i][j][r] - lse.x, kLog2e, less));
          if (mr + 4 * (lane >> 5) == row) d -= 1.f;
          d = live && m0 + mr + 4 * (lane >> 5) < M ? d * ratio : 0.f;
          sum[i * 16 + r] += d;
          // For bf16 inputs d goes to the two products in bf16: they take
          // half the time and traffic that two bf16 parts of it would.  Its
          // roundings (2^-8 of a term at most) are independent; the outputs'
          // own rounding outweighs them: 8192 x 50021 x 2048, error against
          // 64 bits 1.658e-3 for dx and 1.654e-3 for dw, where 32-bit terms
          // rounded once have 1.655e-3 and 1.651e-3.
          if (SA == F32)
            static_cast<float*>(p.out)[at + mr * p.out_ld] = d;
          else
            static_cast<bf16*>(p.out)[at + mr * p.out_ld] = (bf16)d;
        }
    }
    if (p.rowsum) {
      // Each exchange halves the values a lane answers for: after five, lane
      // l holds the sums of values l * MF / 2 and on.
      int lo = 0;
      fold<MF * 8>(sum, 16, lane, lo);
      fold<MF * 4>(sum, 8, lane, lo);
      fold<MF * 2>(sum, 4, lane, lo);
      fold<MF>(sum, 2, lane, lo);
      fold<MF / 2>(sum, 1, lane, lo);
      // one 32 x 32 tile a wave: 16 values, each still in a pair of lanes
      if (MF == 1) sum[0] += __shfl_xor(sum[0], 1, 64);
      constexpr int LEFT = MF / 2 > 0 ? MF / 2 : 1;
      float* out = p.rowsum
          + ((g * p.tiles_n + tn) * H::WN + wave % H::WN) * (long long)M;
#pragma unroll
      for (int i = 0; i < LEFT; ++i) {
        const int v = lo + i;
        const int m = m0 + v / 16 * 32 + acc_row(v % 16, lane);
        if (m < M && (MF > 1 || !(lane & 1))) out[m] = sum[i];
      }
    }
  }
}

// out[g][i] = sum over splits of partial[split][g][i] (+ bias[i % n]), i over
// the m * n outputs of a group; V values a thread.
template <typename T, int V>
__global__ __launch_bounds__(kThreads)
void join_kernel(const float* __restrict__ partial, int splits,
                 long long slab, long long size, long long n, T* out,
                 long long out_group, const T* bias, long long bias_group) {
  const long long g = blockIdx.y;
  const long long step = (long long)gridDim.x * kThreads * V;
  for (long long i = ((long long)blockIdx.x * kThreads + threadIdx.x) * V;
       i < size; i += step) {
    const float* p = partial + g * size + i;
    float s[V];
#pragma unroll
    for (int j = 0; j < V; ++j) s[j] = 0.f;
#pragma unroll 4
    for (int k = 0; k < splits; ++k) {
      float v[V];
      load_n<V>(p + k * slab, v);
#pragma unroll
      for (int j = 0; j < V; ++j) s[j] += v[j];
    }
    if (bias) {
#pragma unroll
      for (int j = 0; j < V; ++j)
        s[j] += to_f(bias[g * bias_group + (i + j) % n]);
    }
    T* o = out + g * out_group + i;
#pragma unroll
    for (int j = 0; j < V; ++j) o[j] = from_f<T>(s[j]);
  }
}

// Merges the vocabulary tiles' (max, sum) of R rows per block, 256 / R threads
// a row, and leaves the block's loss sum and count in 64 bits.  Few rows are
// given more threads each: a thread's tiles come one after another (7 rows,
// 157 tiles: 3.8 us with R = 8 against 7.3 with 32).
template <int R>
__global__ __launch_bounds__(kThreads)
void lse_kernel(const float2* __restrict__ part,
                const float* __restrict__ picked,
                const long long* __restrict__ target, long long ignore,
                long long vocab, int tiles, long long rows,
                float2* __restrict__ lse, float* __restrict__ row_loss,
                double2* __restrict__ sums) {
  constexpr int SEGS = kThreads / R;
  __shared__ float2 seg[SEGS][R];
  const int tl = threadIdx.x % R, sl = threadIdx.x / R;
  const long long g = blockIdx.y;
  for (long long blk = blockIdx.x; blk * R < rows; blk += gridDim.x) {
    const long long n = blk * R + tl;
    float mx = -INFINITY, sum = 0.f;
    if (n < rows) {
      const float2* q = part + g * tiles * rows + n;
#pragma unroll 4
      for (int t = sl; t < tiles; t += SEGS) {
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
        for (int t = 1; t < SEGS; ++t) {
          const float2 v = seg[t][tl];
          const float m = fmaxf(mx, v.x);
          const float ref = m == -INFINITY ? 0.f : m;
          sum = sum * __builtin_amdgcn_exp2f((mx - ref) * kLog2e)
              + v.y * __builtin_amdgcn_exp2f((v.x - ref) * kLog2e);
          mx = m;
        }
        const long long tgt = target[g * rows + n];
        const float l = logf(sum);
        float row = 0.f;
        if (tgt != ignore) {
          const bool word = tgt >= 0 && tgt < vocab;
          if (!word) mx = NAN;
          row = (mx - (word ? picked[g * rows + n] : 0.f)) + l;
          loss = row;
          cnt = 1.0;
        }
        lse[g * rows + n] = make_float2(mx, l);
        row_loss[g * rows + n] = row;
      }
#pragma unroll
      for (int o = R / 2; o > 0; o >>= 1) {
        loss += __shfl_xor(loss, o, R);
        cnt += __shfl_xor(cnt, o, R);
      }
      if (tl == 0 && sums)
        sums[g * ((rows + R - 1) / R) + blk] = make_double2(loss, cnt);
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

// The largest finite magnitude of a group's upstream row gradients, and the
// rows' ratios to it; a row's that is not finite stays its own matter.
__global__ __launch_bounds__(kThreads)
void row_scale_kernel(const float* __restrict__ grad, long long rows,
                      float* __restrict__ top, float* __restrict__ ratio) {
  __shared__ uint32_t red[4];
  const long long g = blockIdx.x;
  uint32_t m = 0;                      // bit patterns order as magnitudes do
  for (long long i = threadIdx.x; i < rows; i += kThreads) {
    const uint32_t b = __float_as_uint(grad[g * rows + i]) & 0x7fffffffu;
    if (b < 0x7f800000u) m = max(m, b);
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1)
    m = max(m, (uint32_t)__shfl_xor((int)m, o, 64));
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = m;
  __syncthreads();
  m = max(max(red[0], red[1]), max(red[2], red[3]));
  const float t = __uint_as_float(m);
  if (threadIdx.x == 0) top[g] = t;
  for (long long i = threadIdx.x; i < rows; i += kThreads) {
    const float v = grad[g * rows + i];
    const bool finite = (__float_as_uint(v) & 0x7fffffffu) < 0x7f800000u;
    ratio[g * rows + i] = !finite ? v : m == 0 ? 0.f : v / t;
  }
}

Op make_op(const Mat& m, bool kmajor, long long rows, long long k) {
  Op o;
  o.p = m.p;
  o.ld = m.ld;
  o.group = m.group;
  o.rows = (int)rows;
  o.ext = (int)(m.padded ? m.ld : kmajor ? rows : k);
  o.e = m.e;
  o.e_ld = m.e_ld;
  o.e_group = m.e_group;
  return o;
}

template <Src SA, bool KMA, Src SB, bool KMB, typename H, Epi E>
void launch_as(Params& p, long long groups, hipStream_t s) {
  p.tiles_m = (int)ceil_div(p.a.rows, H::BM);
  p.tiles_n = (int)ceil_div(p.b.rows, H::BN);
  const dim3 grid((unsigned)(p.tiles_m * p.tiles_n), (unsigned)p.splits,
                  (unsigned)groups);
  gemm_kernel<SA, KMA, SB, KMB, H, E><<<grid, H::THREADS, 0, s>>>(p);
}

template <Src SA, bool KMA, Src SB, bool KMB, Epi E>
void launch(Params& p, long long groups, Size size, hipStream_t s) {
  if (size == LARGE)
    launch_as<SA, KMA, SB, KMB, Large, E>(p, groups, s);
  else if (size == SMALL)
    launch_as<SA, KMA, SB, KMB, Small, E>(p, groups, s);
  else
    launch_as<SA, KMA, SB, KMB, Tiny, E>(p, groups, s);
}

// Tile shape and parts of the contraction, by an estimate of the time.  A
// compute unit works off blocks in rounds: one large, two small (three in
// fp32) or three tiny at once.  A round's time is its area and its depth plus
// a fixed part (filling the pipeline, the epilogue), which a large block alone
// does not hide as well.  Measured: large tiles are 1.16 times as fast in the
// long run (bf16 logits 8192 x 50021 x 2048), small ones 1.1 times on short
// contractions (fp32 logits 16 x 500 x 5000 x 300), tiny ones 2.3 times where
// few blocks would leave units idle (fp32 2048 x 128 x 128, 8 us).
struct Tiling {
  Size size;
  int splits;
};
const int kTileM[3] = {Tiny::BM, Small::BM, Large::BM};
const int kTileN[3] = {Tiny::BN, Small::BN, Large::BN};

// `deep`: whether the contraction may be cut into parts, each at least 256
// deep.  `products`: matrix instructions per multiplication (1, 3 or 6).
Tiling tiling(long long groups, long long m, long long n, long long k,
              bool deep, int products) {
  // the time of a round by the blocks on a compute unit, 0 to 3
  const bool parts = products > 1;
  const int most_blocks[3] = {3, parts ? 3 : 2, 1};
  const double round[3][4] = {{0, 0.5, 0.8, 1.12},
                              {0, 1.5, 2.32, 3.25},
                              {0, 4.0, 0, 0}};
  const double fixed[3] = {60, 50, 92};
  // 128 x 128 x 1 steps of a compute unit per microsecond
  const double rate = products == 6 ? 24 : products == 3 ? 45 : 135;
  const long long most = deep ? std::max<long long>(
      1, std::min<long long>(k / 256, 64)) : 1;
  Tiling best = {SMALL, 1};
  double least = -1;
  for (int z = 0; z < 3; ++z) {
    const long long tiles =
        ceil_div(m, kTileM[z]) * ceil_div(n, kTileN[z]) * groups;
    // tiny tiles of a huge output: too many blocks, and never the best
    if (z == TINY && tiles > 1 << 16) continue;
    for (long long splits = 1; splits <= most; ++splits) {
      const long long blocks = tiles * splits, slots = 256 * most_blocks[z];
      const double rounds = round[z][most_blocks[z]] * (blocks / slots)
          + round[z][ceil_div(blocks % slots, 256)];
      double us = rounds * (ceil_div(k, splits) + fixed[z]) / rate;
      // the parts are written, read and joined
      if (splits > 1) us += 4 + (2 * splits + 1) * 4e-6 * m * n * groups / 4;
      if (least < 0 || us < least) {
        least = us;
        best = {(Size)z, (int)splits};
      }
    }
  }
  return best;
}

int products_of(DType a, bool b_act8) {
  return a != kF32 ? 1 : b_act8 ? 3 : 6;
}

unsigned grid_of(long long blocks) {
  return (unsigned)std::min<long long>(std::max<long long>(blocks, 1),
                                       1 << 20);
}

}  // namespace

int gemm_splits(const Gemm& g) {
  return tiling(g.groups, g.m, g.n, g.k, true,
                products_of(g.ta, g.b.e != nullptr)).splits;
}

void product_tiling(long long groups, long long m, long long n, long long k,
                    bool deep, DType a, bool b_act8, int* tile, int* splits) {
  const Tiling t = tiling(groups, m, n, k, deep, products_of(a, b_act8));
  *tile = kTileM[t.size];
  *splits = t.splits;
}

void gemm(const Gemm& g, hipStream_t s) {
  Params p = {};
  p.a = make_op(g.a, g.a_kmajor, g.m, g.k);
  p.b = make_op(g.b, g.b_kmajor, g.n, g.k);
  p.k = (int)g.k;
  p.splits = g.partial ? g.splits : 1;
  p.out = g.out;
  p.out_ld = g.out_ld;
  p.out_group = g.out_group;
  p.accumulate = g.accumulate;
  p.bias = g.bias;
  p.bias_group = g.bias_group;
  p.partial = g.partial;
  p.scale = g.scale;
  const bool f = g.ta == kF32;
  const Size size = tiling(g.groups, g.m, g.n, g.k, true,
                           products_of(g.ta, g.b.e != nullptr)).size;
  const long long n = g.groups;
  if (g.b.e) {                                     // dY' X8
    if (f) launch<F32, true, ACT8, true, STORE>(p, n, size, s);
    else launch<BF16, true, ACT8, true, STORE>(p, n, size, s);
  } else if (!g.a_kmajor && !g.b_kmajor) {         // X W'
    if (f) launch<F32, false, F32, false, STORE>(p, n, size, s);
    else launch<BF16, false, BF16, false, STORE>(p, n, size, s);
  } else if (!g.a_kmajor) {                        // dY W
    if (f) launch<F32, false, F32, true, STORE>(p, n, size, s);
    else launch<BF16, false, BF16, true, STORE>(p, n, size, s);
  } else {                                         // P' W, P stored by word
    if (f) launch<F32, true, F32, true, STORE>(p, n, size, s);
    else launch<BF16, true, BF16, true, STORE>(p, n, size, s);
  }
}

void join_partials(const float* partial, int splits, long long groups,
                   long long m, long long n, void* out, long long out_group,
                   const void* bias, long long bias_group, DType tout,
                   hipStream_t s) {
  const long long size = m * n, slab = groups * size;
  const bool four = size % 4 == 0;
  const dim3 grid(grid_of(ceil_div(size, kThreads * (four ? 4 : 1))),
                  (unsigned)groups);
#define BLADES_JOIN(T, V)                                                  \
  join_kernel<T, V><<<grid, kThreads, 0, s>>>(                             \
      partial, splits, slab, size, n, static_cast<T*>(out), out_group,     \
      static_cast<const T*>(bias), bias_group)
  if (tout == kF32) {
    if (four) BLADES_JOIN(float, 4); else BLADES_JOIN(float, 1);
  } else {
    if (four) BLADES_JOIN(bf16, 4); else BLADES_JOIN(bf16, 1);
  }
#undef BLADES_JOIN
}

static Size loss_size(const Loss& l) {
  return tiling(l.groups, l.vocab, l.rows, l.dim, false,
                products_of(l.t, false)).size;
}
void loss_tile(const Loss& l, int* m, int* n) {
  *m = kTileM[loss_size(l)];
  *n = kTileN[loss_size(l)];
}
long long loss_row_parts(const Loss& l) {
  const Size z = loss_size(l);
  const int waves = z == LARGE ? Large::WN : z == SMALL ? Small::WN : Tiny::WN;
  return ceil_div(l.rows, kTileN[z]) * waves;
}
static int lse_rows(long long rows) { return rows <= 4096 ? 8 : 32; }
long long loss_sum_blocks(long long rows) {
  return ceil_div(rows, lse_rows(rows));
}

namespace {
Params loss_params(const Loss& l, long long v0, long long nv) {
  Params p = {};
  const long long size = l.t == kF32 ? 4 : 2;
  Mat w = l.w;
  w.p = static_cast<const char*>(w.p) + v0 * w.ld * size;
  p.a = make_op(w, false, nv, l.dim);
  p.b = make_op(l.x, false, l.rows, l.dim);
  p.k = (int)l.dim;
  p.splits = 1;
  p.bias = l.bias ? static_cast<const char*>(l.bias) + v0 * size : nullptr;
  p.bias_group = l.bias_group;
  p.target = l.target;
  p.ignore = l.ignore;
  p.v0 = v0;
  return p;
}
}  // namespace

void loss_forward(const Loss& l, void* part, float* picked, void* lse,
                  float* row_loss, void* block_sums, float* loss,
                  float* count, bool mean, hipStream_t s) {
  Params p = loss_params(l, 0, l.vocab);
  p.part = static_cast<float2*>(part);
  p.picked = picked;
  const Size size = loss_size(l);
  if (l.t == kF32) launch<F32, false, F32, false, LSE>(p, l.groups, size, s);
  else launch<BF16, false, BF16, false, LSE>(p, l.groups, size, s);
  const long long blocks = loss_sum_blocks(l.rows);
  const auto merge = lse_rows(l.rows) == 8 ? lse_kernel<8> : lse_kernel<32>;
  merge<<<dim3(grid_of(blocks), (unsigned)l.groups), kThreads, 0, s>>>(
      p.part, picked, l.target, l.ignore, l.vocab, p.tiles_m, l.rows,
      static_cast<float2*>(lse), row_loss, static_cast<double2*>(block_sums));
  if (loss)
    loss_sum_kernel<<<dim3((unsigned)l.groups), kThreads, 0, s>>>(
        static_cast<const double2*>(block_sums), blocks, loss, count, mean);
}

void loss_logit_grad(const Loss& l, long long v0, long long nv,
                     const void* lse, const float* ratio, void* pt,
                     long long pt_ld, long long pt_group, float* rowsum,
                     hipStream_t s) {
  Params p = loss_params(l, v0, nv);
  p.rowsum = rowsum;
  p.lse = static_cast<const float2*>(lse);
  p.ratio = ratio;
  p.out = pt;
  p.out_ld = pt_ld;
  p.out_group = pt_group;
  const Size size = loss_size(l);
  if (l.t == kF32) launch<F32, false, F32, false, GRAD>(p, l.groups, size, s);
  else launch<BF16, false, BF16, false, GRAD>(p, l.groups, size, s);
}

void row_scale(const float* grad, long long groups, long long rows,
               float* top, float* ratio, hipStream_t s) {
  row_scale_kernel<<<dim3((unsigned)groups), kThreads, 0, s>>>(grad, rows,
                                                               top, ratio);
}

}  // namespace token_ops
