// Shared pieces of the gated delta rule's kernels.
//
//   S_t = a_t S_{t-1} + k_t u_t^T,  a_t = exp(g_t),  u_t = beta_t e_t,  e_t = v_t - a_t S_{t-1}^T k_t,  o_t = scale S_t^T q_t
//
// per value head; value head h reads key head h / (HV / HK).  States are key-major fp32, S[n][h][k][v].
#pragma once

#include "pkda_common.cuh"
#include "pkda_launch.h"

namespace pkda {
namespace gdr {

// Smallest log-decay that a cumulative sum takes in.  exp(-128) is zero in fp32 (the build flushes denormals), so nothing
// that a smaller one would give is lost, while -inf, the way to forget everything at a document's first token, would make
// differences of two sums NaN.  64 tokens at the limit leave sums of 8,192, kept to 48 bits (chunk_scalars).
constexpr float kLeastDecay = -128.f;
// (The order keeps a NaN.)
__device__ __forceinline__ float bounded_decay(float g) { return g < kLeastDecay ? kLeastDecay : g; }

struct Params {
  Geo geo;  // geo.heads: value heads
  int key_heads, group;  // group = value heads per key head
  float scale;
  const void *q, *k, *v;
  const float* g;
  const void* beta;
  bool beta32;  // beta (and its gradient) in fp32 beside bf16 activations
  const float* S0;
};

inline int act_dtype(const pkda_gdr_problem& p) { return p.dtype & ~PKDA_GDR_BETA_F32; }
inline bool beta_in_fp32(const pkda_gdr_problem& p) { return p.dtype != PKDA_BF16; }

// T: the activations' type.  (From L2: see chunk_scalars.)
template <typename T> __device__ __forceinline__ float load_beta(const Params& p, size_t at) {
  if (sizeof(T) == 4 || p.beta32) return __ldcg(static_cast<const float*>(p.beta) + at);
  return to_f(__ldcg(static_cast<const bf16*>(p.beta) + at));
}
template <typename T> __device__ __forceinline__ void store_dbeta(const Params& p, void* dbeta, size_t at, float x) {
  if (sizeof(T) == 4 || p.beta32) static_cast<float*>(dbeta)[at] = x;
  else static_cast<bf16*>(dbeta)[at] = __float2bfloat16(x);
}

// Where sequence n lies.  Offsets of a packed batch come from the caller: whatever they hold, the tokens stay inside the tensors.
// (All but the forward chain without saved buffers read the copy that gdr_offsets_kernel has put in order; chunk0 is only theirs.)
__device__ __forceinline__ SeqInfo sequence(const Geo& g, int n) {
  SeqInfo s = seq_info(g, n);
  if (g.cu_seqlens) {
    const int end = min(s.bos + max(s.len, 0), g.total_tokens);
    s.bos = max(s.bos, 0);
    s.len = max(end - s.bos, 0);
    s.nchunks = (s.len + kChunk - 1) / kChunk;
  }
  return s;
}

// Without saved buffers there is no room for a packed batch's offsets put in order: a CTA of a forward chain takes the largest of the
// offsets up to its own by itself, so that sequences of offsets that run backwards are cut as gdr_offsets_kernel cuts them and no row has
// two writers.  Returns whether `s`, what the sequence's own two offsets say, had to be changed.  (This passes while the state and the
// first rows are on their way.  256 sequences of one token of 32 heads of 128 take 349 us, 362 without; 4,096 of 4 heads of 64 take
// 225 us, 200 without: a CTA reads 2 bytes a sequence beside its states.)
template <int kThreads> __device__ __forceinline__ bool cut_sequence(const Geo& g, int n, SeqInfo& s) {
  if (!g.cu_seqlens || g.chunk_offsets) return false;
  __shared__ int s_max[kThreads / 32];
  const int skip = (int)((16 - reinterpret_cast<uintptr_t>(g.cu_seqlens) % 16) % 16) / 4;  // (four offsets at a time)
  int bos = (int)threadIdx.x < min(skip, n + 1) ? max(g.cu_seqlens[threadIdx.x], 0) : 0, i = skip + 4 * (int)threadIdx.x;
#pragma unroll 4
  for (; i + 3 <= n; i += 4 * kThreads) {
    const int4 c = *reinterpret_cast<const int4*>(g.cu_seqlens + i);
    bos = max(max(max(bos, c.x), max(c.y, c.z)), c.w);
  }
#pragma unroll
  for (int j = 0; j < 3; ++j)
    if (i + j <= n) bos = max(bos, g.cu_seqlens[i + j]);
  bos = __reduce_max_sync(0xffffffffu, bos);
  if ((threadIdx.x & 31) == 0) s_max[threadIdx.x >> 5] = bos;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kThreads / 32; ++w) bos = max(bos, s_max[w]);
  bos = min(bos, g.total_tokens);
  if (bos == s.bos) return false;
  s.bos = bos;
  s.len = min(max(g.cu_seqlens[n + 1], bos), g.total_tokens) - bos;
  s.nchunks = (s.len + kChunk - 1) / kChunk;
  return true;
}

// Cumulative log-decays of a chunk and its betas (`at`: its first token's), by one warp: lane l owns tokens 2 l and 2 l + 1.  Tokens past the end of the
// sequence decay by nothing and write nothing.  The sums are kept to 48 bits, sG + sGlo: what counts are differences of them,
// and 64 tokens of strong decay reach sums of hundreds, whose 24 bits leave differences of 1 with errors of 2^-16.  Both are in
// units of log 2.  Returns the chunk's total, G_L.  (Read from L2: a launch beside another has no wait that would make a line of the
// first level's cache good.)
template <typename T>
__device__ __forceinline__ double chunk_scalars(const Params& p, size_t at, int valid, float* sG, float* sGlo, float* sBeta) {
  const int lane = threadIdx.x & 31, t0 = 2 * lane, heads = p.geo.heads;
  const float* g = p.g + at;
  const double g0 = t0 < valid ? (double)bounded_decay(__ldcg(g + (size_t)t0 * heads)) : 0.0;
  const double g1 = t0 + 1 < valid ? (double)bounded_decay(__ldcg(g + (size_t)(t0 + 1) * heads)) : 0.0;
  sBeta[t0] = t0 < valid ? load_beta<T>(p, at + (size_t)t0 * heads) : 0.f;
  sBeta[t0 + 1] = t0 + 1 < valid ? load_beta<T>(p, at + (size_t)(t0 + 1) * heads) : 0.f;
  constexpr double kLog2eD = 1.4426950408889634074;
  const double x1 = g1 * kLog2eD;
  double run = g0 * kLog2eD + x1;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const double y = __shfl_up_sync(0xffffffffu, run, o);
    if (lane >= o) run += y;
  }
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const double x = j ? run : run - x1;
    sG[t0 + j] = (float)x;
    sGlo[t0 + j] = (float)(x - (double)(float)x);
  }
  return __shfl_sync(0xffffffffu, run, 31);
}
// exp of the difference of two cumulative sums (<= 0 for gates that decay).
__device__ __forceinline__ float decay_between(float hi, float lo, float hi0, float lo0) { return exp2f((hi - hi0) + (lo - lo0)); }

// Chunks of 64 tokens: exact for a dense batch, an upper bound for a packed one.
inline size_t chunk_count(const pkda_gdr_problem& p) {
  if (p.cu_seqlens) return (size_t)p.total_tokens / kChunk + p.n_seqs;
  return (size_t)p.n_seqs * ((p.seq_len + kChunk - 1) / kChunk);
}

// Token-by-token kernels (gdr_recurrent.cu).  e, h: what a backward needs, or NULL.
int exact_forward(const pkda_gdr_problem& p, const Params& base, void* o, float* final_state, float* e, float* h, cudaStream_t st);
int exact_backward(const pkda_gdr_problem& p, const Params& base, const pkda_gdr_bwd_args& a, const float* e, const float* h, float* y,
                   float* dh, cudaStream_t st);

// What other operators on packed batches take from here (gdr_entry.cu): the offsets in order with the first chunk of each sequence,
// and zeros in the rows that no sequence owns.
struct Rows {
  void* ptr[5];
  long long bytes[5];  // of a row; a multiple of 2
};
int launch_offsets(const int* cu, int n_seqs, int total, int* bounds, int* offs, cudaStream_t st);
int launch_unowned_rows(const int* cu, int n_seqs, int total, const Rows& r, cudaStream_t st);

}  // namespace gdr
}  // namespace pkda
