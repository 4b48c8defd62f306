// Launch functions of the token-model operators (layer norm, linear layers
// with a fused loss, 8-bit activation checkpoints).  Plain pointers and a
// stream: the tensor checks live in token_bindings.cpp, the kernels in
// layer_norm.hip, act8.hip and token_gemm.hip.
//
// A "group" is one client of a population trained as one batch: a group owns
// `rows` consecutive rows and its own parameter gradients.  Parameters are
// shared (group stride 0) or one set per group.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

namespace token_ops {

enum DType : int { kF32 = 0, kBF16 = 1 };

inline long long ceil_div(long long a, long long b) { return (a + b - 1) / b; }

// ------------------------------------------------------------- layer_norm
struct NormArgs {
  const void* x;
  const void* dy;     // backward only
  const void* w;      // may be null
  const void* b;      // may be null
  void* y;            // forward: y, backward: dx
  float* mean;
  float* rstd;
  void* dw;           // backward, may be null
  void* db;           // backward, may be null
  float* partial;     // backward workspace,
                      // [groups][norm_partial_blocks()][2][dim]
  long long groups, rows, dim;
  long long w_stride, b_stride;  // elements between groups' parameters
  float eps;
};
long long norm_partial_blocks(long long groups, long long rows, long long dim,
                              DType t);
void norm_forward(const NormArgs& a, DType t, hipStream_t s);
void norm_backward(const NormArgs& a, DType t, hipStream_t s);

// A factor per group: num[g], or num[g] / den[g] (0 where den is 0), or 1
// where num is null.
struct Scale {
  const float* num;
  const float* den;
};

// out[g][c] = scale[g] * sum over blocks of partial[g][block][c]
void join_rows(const float* partial, long long groups, long long blocks,
               long long cols, void* out, long long out_group,
               const Scale& scale, DType t, hipStream_t s);

// Sums over rows: out[g][c] = sum_r x[g][r][c], through a workspace of
// groups * colsum_blocks() * cols floats.
long long colsum_blocks(long long groups, long long rows, long long cols);
void colsum(const void* x, void* out, float* partial, long long groups,
            long long rows, long long cols, DType t, hipStream_t s);

// ------------------------------------------------------------------- act8
// q[rows][dim] int8 and e[rows][ceil(dim/128)]: x ~ q * 2^(e - 127).
void act8_pack(const void* x, int8_t* q, uint8_t* e, long long rows,
               long long dim, DType t, hipStream_t s);
void gelu_forward(const void* x, void* y, int8_t* q, uint8_t* e,
                  long long rows, long long dim, DType t, hipStream_t s);
void gelu_backward(const void* dy, const int8_t* q, const uint8_t* e,
                   void* dx, long long rows, long long dim, DType t,
                   hipStream_t s);

// ------------------------------------------------------- matrix products
struct Mat {              // row-major, `ld` elements between rows
  const void* p;
  long long ld;
  long long group;        // elements between groups (0: shared)
  const uint8_t* e;       // exponents of 8-bit storage, else null
  long long e_ld, e_group;
  bool padded;            // rows may be read, as zeros, up to `ld`
};

// out[g][m][n] = scale[g] * sum_k A[g](m,k) * B[g](n,k) (+ bias[g][n]), sums in
// 32 bits.
//   a_kmajor: A is stored [k][m] instead of [m][k]; likewise b_kmajor.
// With `partial` set and splits > 1 the contraction is cut into `splits`
// parts whose sums go to partial[split][g][m][n] and are joined afterwards;
// `accumulate` keeps adding into `partial` (joined by the caller).
struct Gemm {
  Mat a, b;
  bool a_kmajor, b_kmajor;
  DType ta, tb;           // tb ignored where b.e is set
  long long groups, m, n, k;
  void* out;
  long long out_ld, out_group;
  DType tout;
  const void* bias;
  long long bias_group;
  float* partial;
  int splits;
  bool accumulate;
  Scale scale;
};
// Parts the contraction is best cut into (1: write `out` at once).
int gemm_splits(const Gemm& g);
void gemm(const Gemm& g, hipStream_t s);
// Rows of the square output tile and parts of the contraction that a product
// takes; `deep`: whether it may be cut.  For tests that have to reach each.
void product_tiling(long long groups, long long m, long long n, long long k,
                    bool deep, DType a, bool b_act8, int* tile, int* splits);
// out = sum over splits of partial (+ bias), rounded to tout; a group's rows
// lie without gaps
void join_partials(const float* partial, int splits, long long groups,
                   long long m, long long n, void* out, long long out_group,
                   const void* bias, long long bias_group, DType tout,
                   hipStream_t s);

// ----------------------------------------------- loss of a linear head
struct Loss {
  Mat x;                  // [groups][rows][dim]
  Mat w;                  // [groups or shared][vocab][dim]
  const void* bias;       // [vocab], may be null
  long long bias_group;
  const long long* target;  // [groups][rows]
  long long groups, rows, vocab, dim, ignore;
  DType t;
};
// Tiles the loss is computed in: m words by n rows.
void loss_tile(const Loss& l, int* m, int* n);
// part: [groups][vocabulary tiles][rows] float2; picked: [groups][rows] float.
// Writes lse, a row's largest logit and the logarithm of its sum relative to
// that as float2 [groups][rows] (their sum would round the logarithm away where
// logits are large), and row_loss [groups][rows]; with `loss` set also its sum (or mean) per
// group and the number of counted rows, through block_sums
// [groups][loss_sum_blocks(rows)] double2.
long long loss_sum_blocks(long long rows);
void loss_forward(const Loss& l, void* part, float* picked, void* lse,
                  float* row_loss, void* block_sums, float* loss,
                  float* count, bool mean, hipStream_t s);
// Upstream gradients per row as top[g] * ratio[g][row], |ratio| <= 1.
void row_scale(const float* grad, long long groups, long long rows,
               float* top, float* ratio, hipStream_t s);
// One piece of the vocabulary [v0, v0+nv): pt[g][v][ld] = ratio * (softmax -
// onehot), token-minor, zero beyond rows and nv up to whole tiles.
// The group's upstream factor stays out of it: rounded into the bf16 values
// it would be one relative error, up to 2^-8, common to all of them.
// rowsum (may be null): [groups][loss_row_parts()][nv] sums over rows, before
// any rounding to bf16.
void loss_logit_grad(const Loss& l, long long v0, long long nv,
                     const void* lse, const float* ratio, void* pt,
                     long long pt_ld, long long pt_group, float* rowsum,
                     hipStream_t s);
long long loss_row_parts(const Loss& l);

}  // namespace token_ops
