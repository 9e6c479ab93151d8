// Shared pieces of linear attention with a decay for each head.
//
//   S_t = a_t S_{t-1} + k_t v_t^T,  a_t = exp(g_t),  o_t = scale S_t^T q_t
//
// per value head; value head h reads key head h / (HV / HK); g is a number a token and head or one a head.  States are key-major
// fp32, S[n][h][k][v].
//
// Forward and gradients are one operation.  With reads x, keys y and values z of a state R [y][z], forwards or backwards in time,
//   out_a = c sum_b D_ab (x_a . y_b) z_b + r_a R^T x_a,     R' = decay R + sum_b w_b y_b z_b^T,
// D_ab the decay between the tokens (b not behind a in the direction of time), r_a what R decays by up to a, w_b what token b's
// write decays by up to the end:
//   o  = (x, y, z) = (q, k, v)   forwards            dq = (do, v, k)   forwards, R the transposed state
//   dv = (k, q, do)  backwards, R the cotangent dS of the state                dk = (v, do, q)   backwards, R its transpose
// The scale goes to the reads of the forward passes and to the writes of the backward ones, so that R is always in its own units.
//
// The gate's gradient.  With W_ij = scale D_ij (q_i.k_j)(do_i.v_j) (i reads what j < i wrote; the diagonal has no decay in it) and the
// states in front and behind as further writers and readers, the decay at t takes part in all W_ij with i >= t > j:
//   dg_t = sum_{u >= t} (row_u - col_u) + <S_end, dS_end>,   row_i = sum_{j < i} W_ij,   col_j = sum_{i > j} W_ij
// up to any later token `end`.  row is part of dq.q, col part of dk.k; <S, dS> counts the pairs that reach over the end.
#pragma once

#include "gdr_common.cuh"

namespace pkda {
namespace la {

using gdr::bounded_decay;

// One operation of a call.
struct Pass {
  const void *x, *y, *z, *u;  // u (or NULL): row sums of (out without the token's own write) * u go to `dots`
  int x_group, y_group, z_group, u_group;  // value heads per head of the tensor
  const float* init;          // R at the start (in the direction of time), or NULL: zeros
  float *fin, *fin2;          // R at the end goes there (either may be NULL)
  int init_t, fin_t;          // whether these lie transposed, [z][y]
  void* out;                  // [tokens][heads][D], activations or, with out32, fp32
  int out32;
  float* dots;                // [slices][heads][tokens]
  float c, read, write;       // scale of the pairs, of what is read of R, of what is written to it
  int reverse;
};

struct Call {
  Geo geo;  // geo.heads: value heads
  int group;
  const float* g;
  int g_step;  // heads, or 0 where a head has one decay
};

// The log-decay of (token, head).
__device__ __forceinline__ float gate(const Call& c, size_t token, int h) { return bounded_decay(__ldg(c.g + token * c.g_step + h)); }

// Token by token in fp32 (la_chain.cu).  All passes in one launch.
int launch_chain(const Call& c, int D, int dtype, const Pass* passes, int n, cudaStream_t st);
// Columns of z that one CTA of the chain takes, and so the slices that `dots` has.
int chain_slices(long long units, int D);

// Segments.  Chunks of a sequence go in segments of `chunks` chunks; entry e of a buffer that has something for every segment belongs
// to (sequence, segment), with one such for each head.  Dense batches have n * segs + seg; in a packed one sequence n starts at
// offs[n] / chunks + n, which leaves room for all of its segments whatever the lengths.  chunks = 0: a sequence is one segment.
struct Segments {
  int chunks = 0, segs = 1;   // segments of a sequence of a dense batch
  long long entries = 0;      // a packed batch's: at most
};
__device__ __forceinline__ int first_entry(const Geo& g, const Segments& s, int n) {
  if (!s.chunks) return n;
  return g.cu_seqlens ? g.chunk_offsets[n] / s.chunks + n : n * s.segs;
}
// The (sequence, segment) of an entry; false where there is none.
__device__ __forceinline__ bool find_segment(const Geo& g, const Segments& s, int e, int& n, int& seg) {
  if (!s.chunks || !g.cu_seqlens) {
    n = e / (s.chunks ? s.segs : 1);
    seg = s.chunks ? e - n * s.segs : 0;
    return true;
  }
  int lo = 0, hi = g.n_seqs - 1;  // the last sequence that starts at e or before
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (first_entry(g, s, mid) <= e) lo = mid; else hi = mid - 1;
  }
  n = lo;
  seg = e - first_entry(g, s, lo);
  const int len = g.cu_seqlens[n + 1] - g.cu_seqlens[n], chunks = (len + kChunk - 1) / kChunk;
  return seg < max((chunks + s.chunks - 1) / s.chunks, 1);
}

// dg from rows and columns (a segment at a time).
struct GateGrad {
  Call c;
  Segments segments;
  const float *row, *col;  // [slices][heads][tokens]
  int row_slices, col_slices;
  const float* X;          // [entries][heads][x_parts]: <S, dS> at the end of a segment in parts; or NULL: formed here from S and dS (either may be NULL: 0)
  int x_parts;
  const float *S, *dS;
  const float *S0, *dS0;   // with X: the same product at a sequence's start (S0 NULL: 0; dS0 NULL beside S0: not known)
  int D;
  float* dg;               // [tokens][heads], or NULL
  double* part;            // [entries][heads], or NULL
  float* dg_head;          // [heads]
};
int launch_gate_grad(const GateGrad& a, cudaStream_t st);

// out[token][hk][:] = sum over the group of part[token][h][:]
int launch_group_sum(const float* part, void* out, int dtype, long long tokens, int key_heads, int group, int D, cudaStream_t st);

}  // namespace la
}  // namespace pkda
