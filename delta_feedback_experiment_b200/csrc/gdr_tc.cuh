// The chunked gated delta rule on tcgen05 (bf16, heads of 128 channels, chunks of 64 tokens).
//
// Per (chunk, value head), with G the cumulative log-decay, D_ij = exp(G_i - G_j) for i >= j, s the query scale, S the state
// at the chunk's start:
//   M = tril(D * k k^T, -1)     P = s tril(D * q k^T)     N = (I + M diag b)^-1 M     T = I - N diag b
//   e = T (v - exp(G) k S)      u = b e      o = s exp(G) q S + P u      S' = exp(G_L) S + (exp(G_L - G) k)^T u
// and backwards, from the cotangents do and dS':
//   du = exp(G_L - G) k dS' + P^T do     y = du - N^T (b du)     dv = b y     dS = exp(G_L) dS' + (s exp(G) q)^T do - (exp(G) k)^T dv
// (T = (I + M diag b)^-1 and I - diag(b) N = (I + diag(b) M)^-1: one N serves both, and b = 0 needs no division: db = e.y.)
// Every factor is a decay between two tokens, at most 1, so no gate needs a case of its own; the decay is a number per
// token and head, so it scales rows and columns of accumulators where PKDA's has to go into the operands.
#pragma once

#include "gdr_common.cuh"
#include "pkda_tc.cuh"

namespace pkda {
namespace gdr {

constexpr int kW = 128;            // head width of the chunked kernels
// fp32 per (chunk, value head), 64 each: exp(G), beta, exp(G_L - G) beta, exp(G_L - G) (the scans'), then G in units of log 2, hi and lo.
constexpr int kScanScalars = 4 * 64, kScalars = 6 * 64;

// Precision.  q, k, v, do are bf16 and enter the products as they are.  What the chain of the states is made of (T, P, S, the
// corrections and writes) is computed, and a bf16 operand of it would leave the states and the gate's gradient, which are fp32,
// with errors of 2^-9.  So such an operand is split, x = hi + lo with hi = bf16(x), lo = bf16(x - hi), off by at most 2^-18 of
// x, and a product takes two passes (three where both sides are split; lo lo is below 2^-18 of it).  The tensor cores have the
// time: a chunk of the scan is bound by its round trips and its bytes.  (Most of what is left in a state, 2.5e-6 of its root mean square,
// comes from the writes of the last tokens.  Three parts of them leave 3.6e-7, 1.2e-6 where the gates hardly decay, and cost the
// chain of a chunk 12 % of its time, 28 % with saved states: not taken.)
//
// What the pair kernel leaves per (chunk, value head), and the states.
struct ChunkBuffers {
  bf16* T;   // [chunk][head][2][8 octets of j][64 i][8], hi and lo
  bf16* T2;  // the same of -diag(b) N (for the backward, or NULL)
  bf16* P;   // the same
  float* scal;   // [chunk][head][kScalars]
  bf16 *e, *h;   // [chunk][head][2][8 token octets][128 v][8], [chunk][head][2][16 key octets][128 v][8] (for the backward, or NULL)
  int* status;   // not zero: a wait of the call's kernels gave up, results are marked with NaN (mark_failed)
};

// Two values to a word of hi parts and one of lo parts.  hi is rounded by integer arithmetic (nearest, ties away from zero),
// which runs at full rate; conversions do not, and the chain of the scan waits for them.  A NaN may lose its hi part: its lo is
// NaN still.  (An infinity becomes a NaN.)
__device__ __forceinline__ void split2(float a, float b, uint32_t& hi, uint32_t& lo) {
  const uint32_t ra = __float_as_uint(a) + 0x8000u, rb = __float_as_uint(b) + 0x8000u;
  hi = __byte_perm(ra, rb, 0x7632);
  lo = pack_bf16(a - __uint_as_float(ra & 0xffff0000u), b - __uint_as_float(rb & 0xffff0000u));
}

__device__ __forceinline__ void mbar_arrive(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}

// One arrival of a warp that has read shared memory which an asynchronous copy writes next.  A load only has to be issued in
// front of an arrival, its value may come later, and with sixteen warps in the queue to shared memory it can come after the copy
// has begun: <S, dS'> read part of the next head's state in 139 of 1,000 calls (2 x 333 tokens, 6 value heads on 2 key heads).
// So which lane arrives depends on what was loaded: `seen` has to be computed from all of a lane's loads.
__device__ __forceinline__ void arrive_behind_loads(uint32_t bar, uint32_t seen) {
  const int who = __any_sync(0xffffffffu, seen == 0x7f800001u);  // (0 or 1; either will do)
  if ((int)(threadIdx.x & 31) == who) mbar_arrive(bar);
}

// Rows `valid` .. 63 of a tile of two swizzled blocks [64 rows][64 channels], `pitch` bytes apart, to zero, by one warp.
// (They hold the next sequence's tokens: a masked product would still let its NaN through.)
__device__ __forceinline__ void zero_rows(unsigned char* tile, int pitch, int valid) {
  for (int i = threadIdx.x & 31; i < (kChunk - valid) * 16; i += 32) {
    const int r = valid + (i >> 4), pc = i & 15;
    *reinterpret_cast<uint4*>(tile + (pc >> 3) * pitch + r * 128 + ((pc & 7) << 4)) = make_uint4(0, 0, 0, 0);
  }
}

// NaN into `count` results, by one warp.
__device__ __forceinline__ void mark_failed(float* at, int count) {
  for (int i = threadIdx.x & 31; i < count; i += 32) at[i] = __int_as_float(0x7fc00000);
}
__device__ __forceinline__ void mark_failed(bf16* at, int count) {
  for (int i = threadIdx.x & 31; i < count; i += 32) at[i] = __float2bfloat16(__int_as_float(0x7fc00000));
}

// What the reverse scan leaves for the gradients: dS' and y per (chunk, value head), laid out like h and e.
struct GradBuffers {
  bf16 *dh, *y;
};

// The chunks [c0, c1) of every sequence of a dense batch, or with c1 = 0 all chunks of any batch.  A launch `beside` the one in
// front of it needs nothing of that (pkda_common.cuh): it does not wait for it at its start, and one of its CTAs does at its end.  The
// scan in front of it is an `ordinary` launch, so that what earlier launches left is complete and visible.
struct Part {
  int c0 = 0, c1 = 0;
  bool beside = false, ordinary = false;
};
__host__ __device__ inline int part_chunks(const Geo& g, const Part& t) { return t.c1 ? g.n_seqs * (t.c1 - t.c0) : g.total_chunks; }
__device__ __forceinline__ int part_chunk(const Geo& g, const Part& t, int x) {  // the x-th of them
  if (!t.c1) return x;
  const int n = x / (t.c1 - t.c0);
  return n * g.chunks_per_seq + t.c0 + x - n * (t.c1 - t.c0);
}
__device__ __forceinline__ SeqInfo part_sequence(const Geo& g, const Part& t, int n) {
  SeqInfo s = sequence(g, n);
  if (t.c1) {
    s.bos += t.c0 * kChunk;
    s.len = min(s.len, t.c1 * kChunk) - t.c0 * kChunk;
    s.chunk0 += t.c0;
    s.nchunks = t.c1 - t.c0;
  }
  return s;
}

int launch_pairs(const Params& p, const ChunkBuffers& b, const Part& part, cudaStream_t st);
int launch_scan(const Params& p, const ChunkBuffers& b, const Part& part, const float* S0, bf16* o, float* ST, cudaStream_t st);
int launch_scan_bwd(const Params& p, const ChunkBuffers& b, const GradBuffers& g, const Part& part, const bf16* d_o, const float* dST, bf16* dv,
                    float* dS0, cudaStream_t st);
int launch_grad(const Params& p, const ChunkBuffers& b, const GradBuffers& g, const Part& part, const bf16* d_o, bf16* dq, bf16* dk, float* dg,
                void* dbeta, cudaStream_t st);

// e, y, h and dS' are written by threads that hold a value channel each.  With octets outermost a warp's store of 16 bytes a
// thread is 512 contiguous bytes; [128 v][..] rows cost 32 sectors of 32 lines a store, 1.9 us of a chunk's step.  They are read
// by plain bulk copies as operand tiles without swizzle (octet_desc).
constexpr int kOctet = kW * 8;     // elements from one octet to the next
__device__ __forceinline__ uint64_t octet_desc(uint32_t tile, int kk) {  // k-step kk: value channels 16 kk ..
  return tc::desc_mnmajor_plain(tile + kk * 256, 128, kOctet * 2);
}

// The pair matrices likewise, octets of columns outermost, written by a thread per row: as an operand with the columns along K
// (k-step kk: columns 16 kk ..) and with the rows along K (rows 16 kk ..).
__device__ __forceinline__ uint64_t pair_desc(uint32_t tile, int kk) { return tc::desc_kmajor_plain(tile + kk * 2048, 1024, 128); }
__device__ __forceinline__ uint64_t pair_desc_t(uint32_t tile, int kk) { return tc::desc_mnmajor_plain(tile + kk * 256, 128, 1024); }

// Tensor map of a [tokens][heads][128] activation in boxes of 64 channels x 64 tokens of one head.
bool map_rows(CUtensorMap* m, const void* base, int heads, int tokens);

}  // namespace gdr
}  // namespace pkda
