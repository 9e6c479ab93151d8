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

// Log-decays add up in fixed point, whole numbers of 2^-40 in units of log 2: sums and differences are exact, whatever their order, and
// 64 bits do in two instructions what fp64 takes far longer for.  64 tokens at the least decay reach 2^54.
constexpr int kFixed = 40;
__device__ __forceinline__ long long to_fixed(float g) {  // g log2(e), whose product is kept to 48 bits
  constexpr float kHi = 1.44269502162933349609375f, kLo = 1.925963033500011079e-8f;
  const float hi = g * kHi, lo = fmaf(g, kHi, -hi) + g * kLo;
  return __float2ll_rn(hi * 1099511627776.f) + __float2ll_rn(lo * 1099511627776.f);
}
__device__ __forceinline__ float2 from_fixed(long long x) {  // in two parts
  const int top = (int)(x >> 24);
  const float hi = (float)top;
  return f2(hi * 1.52587890625e-5f, (float)(int)(x - ((long long)__float2int_rn(hi) << 24)) * 9.094947017729282e-13f);
}
__device__ __forceinline__ float exp2_fixed(long long x) {
  const int w = (int)(x >> kFixed);
  const float e = exp2f((float)(unsigned)(x >> (kFixed - 32)) * 2.3283064365386963e-10f);
  return w < -126 ? 0.f : e * __int_as_float((min(w, 128) + 127) << 23);  // (2^128 is infinity)
}
// 2^x to 2^-27.5 of it (2^-30 in the mean), in two parts: 2^(i / 32) by table, the rest, at most 1/32, by its series (the table-driven
// method of Tang, 1989).  Above 2^-60 the first part is cut off instead of rounded and the second is not zero, so that an infinite
// state times both is infinite still.
static __constant__ float2 kExp2Table[32] = {
    {0x1.0000000000000p+0f, 0x0.0p+0f}, {0x1.059b0e0000000p+0f, -0x1.9d4f520000000p-25f}, {0x1.0b55860000000p+0f, 0x1.9f31220000000p-25f}, {0x1.11301e0000000p+0f, -0x1.fdb4960000000p-25f},
    {0x1.172b840000000p+0f, -0x1.c157420000000p-27f}, {0x1.1d48740000000p+0f, -0x1.d2e8ca0000000p-25f}, {0x1.2387a60000000p+0f, 0x1.ceac480000000p-25f}, {0x1.29e9e00000000p+0f, -0x1.5c04240000000p-25f},
    {0x1.306fe00000000p+0f, 0x1.4636e20000000p-25f}, {0x1.371a740000000p+0f, -0x1.18aac60000000p-25f}, {0x1.3dea640000000p+0f, 0x1.8246840000000p-25f}, {0x1.44e0860000000p+0f, 0x1.8624b40000000p-30f},
    {0x1.4bfdae0000000p+0f, -0x1.593abc0000000p-25f}, {0x1.5342b60000000p+0f, -0x1.2c56100000000p-25f}, {0x1.5ab07e0000000p+0f, -0x1.5bd5ec0000000p-27f}, {0x1.6247ec0000000p+0f, -0x1.f8b5500000000p-25f},
    {0x1.6a09e60000000p+0f, 0x1.9fcef40000000p-26f}, {0x1.71f75e0000000p+0f, 0x1.1d8bee0000000p-25f}, {0x1.7a11480000000p+0f, -0x1.829fd00000000p-25f}, {0x1.82589a0000000p+0f, -0x1.accc7c0000000p-26f},
    {0x1.8ace540000000p+0f, 0x1.15506e0000000p-27f}, {0x1.93737c0000000p+0f, -0x1.e647440000000p-25f}, {0x1.9c49180000000p+0f, 0x1.51f8480000000p-27f}, {0x1.a5503c0000000p+0f, -0x1.b83b540000000p-25f},
    {0x1.ae89fa0000000p+0f, -0x1.a94b140000000p-26f}, {0x1.b7f7700000000p+0f, -0x1.a094380000000p-25f}, {0x1.c199be0000000p+0f, -0x1.3d56b20000000p-27f}, {0x1.cb720e0000000p+0f, -0x1.8837cc0000000p-27f},
    {0x1.d5818e0000000p+0f, -0x1.822dbc0000000p-27f}, {0x1.dfc9740000000p+0f, -0x1.908c940000000p-25f}, {0x1.ea4afa0000000p+0f, 0x1.52486c0000000p-27f}, {0x1.f507660000000p+0f, -0x1.246eb00000000p-26f}};
__device__ __forceinline__ float2 exp2_fixed_two(long long x) {
  const int w = (int)(x >> kFixed);
  if (w < -126) return f2(0.f, 0.f);
  const float2 t = kExp2Table[(int)(x >> (kFixed - 5)) & 31];
  const float r = (float)(unsigned)((x >> (kFixed - 37)) & 0xffffffffu) * (2.3283064365386963e-10f / 32.f * 0.693147180559945f);
  const float s = r * fmaf(r, fmaf(r, fmaf(r, 1.f / 24.f, 1.f / 6.f), 0.5f), 1.f);  // e^r - 1
  const bool up = w >= -60;  // (further down the second part leaves fp32's range, and the first has to be the nearest number)
  const float add = fmaf(t.x, s, t.y), hi = up ? __fadd_rd(t.x, add) : t.x + add, lo = fmaxf(add - (hi - t.x), up ? 0x1p-64f : -1.f);
  const float scale = __int_as_float((min(w, 128) + 127) << 23);
  return f2(hi * scale, w > 127 ? lo : lo * scale);
}

// A value that the compiler keeps: what it reads of the launch's arguments at an index that it does not know it would read again and
// again, at the latency of an indexed constant each time.
__device__ __forceinline__ int kept(int x) {
  asm volatile("" : "+r"(x));
  return x;
}
__device__ __forceinline__ float kept(float x) {
  asm volatile("" : "+f"(x));
  return x;
}
template <typename T> __device__ __forceinline__ T* kept(T* x) {
  asm volatile("" : "+l"(x));
  return x;
}

// One operation of a call.
struct Pass {
  const void *x, *y, *z, *u;  // u (or NULL): row sums of (out without the token's own write) * u go to `dots`
  int x_group, y_group, z_group, u_group;  // value heads per head of the tensor
  const float* init;          // R at the start (in the direction of time), or NULL: zeros
  float* fin;                 // R at the end goes there, or NULL
  int init_t, fin_t;          // whether these lie transposed, [z][y]
  void* out;                  // [tokens][heads][D], activations or, with out32, fp32
  int out32;
  float* dots;                // [slices][heads][tokens]
  float c, read, write;       // scale of the pairs, of what is read of R, of what is written to it
  int reverse;
};

struct Call {
  Geo geo;  // geo.heads: value heads
  const float* g;
  int g_step;  // heads, or 0 where a head has one decay
};

// The log-decay of (token, head), a NaN as it is.  At 128 its exponential is infinite already; sums of what is larger would leave 64 bits.
constexpr float kMostGate = 128.f;
__device__ __forceinline__ float gate(const Call& c, size_t token, int h) {
  const float g = __ldg(c.g + token * c.g_step + h);
  return g > kMostGate ? kMostGate : bounded_decay(g);
}

// One or two tokens forwards, no state but the last (la_chain.cu), where takes_step() says so.
bool takes_step(const Call& c, int D);
int launch_step(const Call& c, int D, int dtype, const Pass& p, cudaStream_t st);
// Columns of z that one CTA of the chain takes, and so the slices that `dots` has, and the parts of an X (a warp each).
int chain_slices(long long units, int D);
int chain_x_parts(long long units, int D);

// Segments.  Chunks of a sequence go in segments of `chunks` chunks; entry e of a buffer that has something for every segment belongs
// to (sequence, segment), with one such for each head.  Dense batches have n * segs + seg; in a packed one sequence n starts at
// offs[n] / chunks + n, which leaves room for all of its segments whatever the lengths.
struct Segments {
  int chunks = 1, segs = 1;   // segments of a sequence of a dense batch
  long long entries = 0;      // a packed batch's: at most
};
__device__ __forceinline__ int first_entry(const Geo& g, const Segments& s, int n) {
  return g.cu_seqlens ? g.chunk_offsets[n] / s.chunks + n : n * s.segs;
}
// The (sequence, segment) of an entry; false where there is none.
__device__ __forceinline__ bool find_segment(const Geo& g, const Segments& s, int e, int& n, int& seg) {
  if (!g.cu_seqlens) {
    n = e / s.segs;
    seg = e - n * s.segs;
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

// Token by token in fp32 (la_chain.cu).  All passes in one launch.  What they leave or take at the segments' ends:
struct ChainEnds {
  Segments segments;
  float* ends = nullptr;            // [entries][heads] the first pass's states (forwards)
  const float* X_states = nullptr;  // those, and <them, R> of the last pass (backwards, R in the order of the states)
  float* X = nullptr;               // [entries][heads][chain_x_parts]
};
int launch_chain(const Call& c, int D, int dtype, const Pass* passes, int n, const ChainEnds& ends, cudaStream_t st);

// dg from rows and columns (a segment at a time).
struct GateGrad {
  Call c;
  Segments segments;
  const float *row, *col;  // [slices][heads][tokens]
  int row_slices, col_slices;
  const float* X;          // [entries][heads][x_parts]: <S, dS> at the end of a segment in parts
  int x_parts;
  const int* grows;        // [entries][heads]: whether a segment has a decay above 1; NULL behind the token-by-token kernels
  const float *S0, *dS0;   // the same product at a sequence's start (S0 NULL: 0; dS0 NULL beside S0: not known)
  int D;
  float* dg;               // [tokens][heads], or NULL
  double* part;            // [entries][heads], or NULL
  float* dg_head;          // [heads]
};
int launch_gate_grad(const GateGrad& a, cudaStream_t st);

// out[token][hk][:] = sum over the group of part[token][h][:], of two tensors
int launch_group_sum(const float* part0, void* out0, const float* part1, void* out1, int dtype, long long tokens, int key_heads, int group, int D,
                     cudaStream_t st);

}  // namespace la
}  // namespace pkda
