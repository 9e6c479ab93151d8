// Gated delta rule, token by token, in fp32: the decoding step, short prompts, and the forward and backward of fp32
// activations and of head widths other than 128.
//
// Forward chain.  The value columns of a state are independent, so a CTA takes 16 to 64 columns of one (sequence, value head) and
// eight (at 16 and 8 channels four and two) adjacent lanes share one, two or four columns, each with its part of the keys in
// registers, two values to a word pair.  Both products of a token are taken on the state before it,
//   e = v - a (S^T k),   o = scale (a (S^T q) + (q.k) beta e),   S <- a S + k (beta e),
// so that a token costs one round of shuffles instead of two; its keys are asked for a token ahead.  Rows of 16 tokens at a
// time are staged in shared memory while the block before is worked on.  What bounds it is a token's chain: half the products
// (in two sums), three shuffles, the correction, the update.  16 states of 128 channels: 9 us for 48 tokens, 0.19 us each; 64
// states, where the packed arithmetic fills the issue slots: 20 us.
//
// Reverse chain, on the cotangent dS of S_t, with the same split:
//   dS += scale q do^T,   y = dS^T k,   dS <- a (dS - k (beta y)^T),   dv = beta y,   dbeta = e.y.
//
// The gradients that need no chain follow per chunk of 64 tokens, in parallel, from e, y and the states S at a chunk's start
// and dS' at its end (G cumulative log-decay, D_ij = exp(G_i - G_j), s = scale):
//   Cq_ij = s beta_j D_ij (do_i.e_j)  (i >= j),   Cm_ij = -beta_i beta_j D_ij (y_i.e_j)  (i > j)
//   dq = Cq k + s exp(G) (S do),   dk = Cq^T q + (Cm + Cm^T) k - exp(G) beta (S y) + exp(G_L - G) beta (dS' e)
//   dG = rows - columns of (Cq * q k^T + Cm * k k^T) + the state parts of dq.q and dk.k, dg = reverse cumulative sum of dG.
// Every factor is at most 1, whatever the gate.
#include "gdr_common.cuh"

#include <type_traits>

namespace pkda {
namespace gdr {

// --------------------------------------------------------------------------- one or two tokens on a cached state
// One CTA holds the whole state of a (sequence, value head) in registers: 128 columns are 32 lanes of four, a warp reads whole
// rows.  Every load of the step is issued before the first use, the state passes through HBM once in each direction: 8,192 states of
// 128 x 128 take 162 us, 1.02 of what their bytes need at the copy rate.
template <int D> struct FewCfg {
  static constexpr int kVQ = D / 4;                                      // lanes of a row
  static constexpr int kKW = 256 / kVQ < D ? 256 / kVQ : D;              // row groups
  static constexpr int kR = D / kKW;                                     // rows of a thread
  static constexpr int kActive = kVQ * kKW;
  static constexpr int kThreads = kActive < 32 ? 32 : kActive;
};

struct RecurrentParams {
  Params p;
  void* o;
  float* ST;
};

template <int D, typename T>
__global__ void __launch_bounds__(FewCfg<D>::kThreads, D == 128 ? 2 : 1) gdr_few_kernel(const RecurrentParams r) {
  after_previous();
  using Cfg = FewCfg<D>;
  constexpr int VQ = Cfg::kVQ, KW = Cfg::kKW, R = Cfg::kR;
  const Params& p = r.p;
  const int H = p.geo.heads, n = blockIdx.x / H, h = blockIdx.x - n * H, hk = h / p.group;
  const SeqInfo sq = sequence(p.geo, n);
  const int tid = threadIdx.x, kq = tid / VQ, vq = tid - kq * VQ;
  const bool active = tid < Cfg::kActive;
  __shared__ float s_k[D], s_q[D], s_qk[8];
  __shared__ __align__(16) float s_ks[KW][D], s_qs[KW][D];
  float4 S[R];
  const size_t sbase = (size_t)blockIdx.x * D * D;
  if (active) {
#pragma unroll
    for (int i = 0; i < R; ++i)
      S[i] = p.S0 ? *reinterpret_cast<const float4*>(p.S0 + sbase + (size_t)(kq * R + i) * D + 4 * vq)
                  : make_float4(0.f, 0.f, 0.f, 0.f);
  }
  for (int t = 0; t < sq.len; ++t) {
    const size_t tok = (size_t)sq.bos + t;
    const size_t key = (tok * p.key_heads + hk) * D, val = (tok * H + h) * D, sc = tok * H + h;
    float qv = 0.f, kv = 0.f;
    if (tid < D) {
      qv = to_f(static_cast<const T*>(p.q)[key + tid]);
      kv = to_f(static_cast<const T*>(p.k)[key + tid]);
    }
    float v[4] = {0.f, 0.f, 0.f, 0.f};
    if (active) {
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = to_f(static_cast<const T*>(p.v)[val + 4 * vq + j]);
    }
    const float a = expf(p.g[sc]), b = load_beta<T>(p, sc);
    if (tid < D) {
      s_q[tid] = qv;
      s_k[tid] = kv;
    }
    float d = qv * kv;
#pragma unroll
    for (int o = 16; o; o >>= 1) d += __shfl_xor_sync(0xffffffffu, d, o);
    if ((tid & 31) == 0 && tid < D) s_qk[tid >> 5] = d;
    __syncthreads();
    if (active) {
      float4 ks = make_float4(0.f, 0.f, 0.f, 0.f), qs = ks;
#pragma unroll
      for (int i = 0; i < R; ++i) {
        const float kk = s_k[kq * R + i], qq = s_q[kq * R + i];
        ks.x += kk * S[i].x; ks.y += kk * S[i].y; ks.z += kk * S[i].z; ks.w += kk * S[i].w;
        qs.x += qq * S[i].x; qs.y += qq * S[i].y; qs.z += qq * S[i].z; qs.w += qq * S[i].w;
      }
      *reinterpret_cast<float4*>(&s_ks[kq][4 * vq]) = ks;
      *reinterpret_cast<float4*>(&s_qs[kq][4 * vq]) = qs;
    }
    __syncthreads();
    if (active) {
      float u[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int w = 0; w < KW; ++w) {
        const float4 x = *reinterpret_cast<const float4*>(&s_ks[w][4 * vq]);
        u[0] += x.x; u[1] += x.y; u[2] += x.z; u[3] += x.w;
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) u[j] = b * (v[j] - a * u[j]);
#pragma unroll
      for (int i = 0; i < R; ++i) {
        const float kk = s_k[kq * R + i];
        S[i].x = a * S[i].x + kk * u[0];
        S[i].y = a * S[i].y + kk * u[1];
        S[i].z = a * S[i].z + kk * u[2];
        S[i].w = a * S[i].w + kk * u[3];
        if (t + 1 == sq.len && r.ST)
          *reinterpret_cast<float4*>(r.ST + sbase + (size_t)(kq * R + i) * D + 4 * vq) = S[i];
      }
      if (kq == 0) {
        float qk = 0.f;
#pragma unroll
        for (int w = 0; w < (D + 31) / 32; ++w) qk += s_qk[w];
        float o[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < KW; ++w) {
          const float4 x = *reinterpret_cast<const float4*>(&s_qs[w][4 * vq]);
          o[0] += x.x; o[1] += x.y; o[2] += x.z; o[3] += x.w;
        }
#pragma unroll
        for (int j = 0; j < 4; ++j)
          static_cast<T*>(r.o)[val + 4 * vq + j] = from_f<T>(p.scale * (a * o[j] + qk * u[j]));
      }
    }
    __syncthreads();
  }
  if (sq.len <= 0 && r.ST && active) {  // an empty sequence hands its state on
#pragma unroll
    for (int i = 0; i < R; ++i) *reinterpret_cast<float4*>(r.ST + sbase + (size_t)(kq * R + i) * D + 4 * vq) = S[i];
  }
}

// --------------------------------------------------------------------------------------------- the chains
// The kernels from here on do not let the next launch start early: its CTAs took what room there was, two on an SM beside idle
// ones, and a chain has to last as long as the fullest SM (fp32, 4 x 512 tokens of 16 heads of 128, forward and backward: 1,157 us
// with an early start, 900 without).
constexpr int kBlock = 16;  // tokens staged at a time
template <int D, int P> struct ChainCfg {              // P: neighbouring columns that a lane has its rows of
  static constexpr int kCols = D < 16 ? D : 16 * P;    // columns of a CTA
  static constexpr int kLanes = D >= 32 ? 8 : D / 4;   // lanes of a column
  static constexpr int kRows = D / kLanes;             // rows of a lane
  static constexpr int kThreads = kCols / P * kLanes < 32 ? 32 : kCols / P * kLanes;
  static constexpr int kGroups = D / kCols;
  // A lane's rows, padded so that the lanes of a column read other banks (a multiple of 4 floats that is odd in those).
  static constexpr int kLd = kRows + (kRows / 4 % 2 ? 0 : 4);
  static constexpr int kRow = kLanes * kLd;
};

// Shared memory of one staged block.
template <int D, int P> struct ChainBlock {
  float k[kBlock][ChainCfg<D, P>::kRow], q[kBlock][ChainCfg<D, P>::kRow];
  float val[kBlock][ChainCfg<D, P>::kCols];            // v, or the output's cotangent
  float a[kBlock], beta[kBlock], qk[kBlock];
};

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

// What a thread holds of the block on its way into shared memory, four values at a time.
__device__ __forceinline__ uint2 load4(const bf16* p) { return *reinterpret_cast<const uint2*>(p); }
__device__ __forceinline__ float4 load4(const float* p) { return *reinterpret_cast<const float4*>(p); }
__device__ __forceinline__ float4 widen4(uint2 r) {
  const float2 a = unpack_bf16(r.x), b = unpack_bf16(r.y);
  return make_float4(a.x, a.y, b.x, b.y);
}
__device__ __forceinline__ float4 widen4(float4 r) { return r; }
template <typename T> struct Four { using Raw = uint2; };
template <> struct Four<float> { using Raw = float4; };

template <int D, int P, typename T> struct ChainLoad {
  using Cfg = ChainCfg<D, P>;
  using Raw = typename Four<T>::Raw;
  static constexpr int kKeys = (kBlock * D / 4 + Cfg::kThreads - 1) / Cfg::kThreads;
  static constexpr int kVals = (kBlock * Cfg::kCols / 4 + Cfg::kThreads - 1) / Cfg::kThreads;
  Raw q[kKeys], k[kKeys], val[kVals];
  float g, beta;

  // Tokens [t0, t0 + 16) of the sequence; those at or past `len` are not read.
  __device__ __forceinline__ void fetch(const Params& p, const void* values, const SeqInfo& sq, int t0, int h, int hk, int col0) {
    const int tid = threadIdx.x;
#pragma unroll
    for (int i = 0; i < kKeys; ++i) {
      const int at = (tid + i * Cfg::kThreads) * 4, t = at / D, c = at % D;
      q[i] = k[i] = Raw{};
      if (t < kBlock && t0 + t < sq.len) {
        const size_t src = ((size_t)(sq.bos + t0 + t) * p.key_heads + hk) * D + c;
        q[i] = load4(static_cast<const T*>(p.q) + src);
        k[i] = load4(static_cast<const T*>(p.k) + src);
      }
    }
#pragma unroll
    for (int i = 0; i < kVals; ++i) {
      const int at = (tid + i * Cfg::kThreads) * 4, t = at / Cfg::kCols, c = at % Cfg::kCols;
      val[i] = Raw{};
      if (t < kBlock && t0 + t < sq.len)
        val[i] = load4(static_cast<const T*>(values) + ((size_t)(sq.bos + t0 + t) * p.geo.heads + h) * D + col0 + c);
    }
    g = beta = 0.f;
    if (tid < kBlock && t0 + tid < sq.len) {
      const size_t at = (size_t)(sq.bos + t0 + tid) * p.geo.heads + h;
      g = p.g[at];
      beta = load_beta<T>(p, at);
    }
  }

  __device__ __forceinline__ void store(ChainBlock<D, P>& s) const {
    const int tid = threadIdx.x;
#pragma unroll
    for (int i = 0; i < kKeys; ++i) {
      const int at = (tid + i * Cfg::kThreads) * 4, t = at / D, c = at % D;
      if (t < kBlock) {
        const int where = c / Cfg::kRows * Cfg::kLd + c % Cfg::kRows;
        *reinterpret_cast<float4*>(&s.q[t][where]) = widen4(q[i]);
        *reinterpret_cast<float4*>(&s.k[t][where]) = widen4(k[i]);
      }
    }
#pragma unroll
    for (int i = 0; i < kVals; ++i) {
      const int at = (tid + i * Cfg::kThreads) * 4, t = at / Cfg::kCols, c = at % Cfg::kCols;
      if (t < kBlock) *reinterpret_cast<float4*>(&s.val[t][c]) = widen4(val[i]);
    }
    if (tid < kBlock) {
      s.a[tid] = expf(g);
      s.beta[tid] = beta;
    }
  }
};

// Sums over the lanes of a column, of several values at a time: a round of each before the next round of any (shuffles stay in
// the order in which they are written, one value after the other would wait three times for each).
template <int D, int N> __device__ __forceinline__ void lanes_sum(float (&x)[N]) {
#pragma unroll
  for (int o = 1; o < ChainCfg<D, 1>::kLanes; o <<= 1) {
    float y[N];
#pragma unroll
    for (int j = 0; j < N; ++j) y[j] = __shfl_xor_sync(0xffffffffu, x[j], o);
#pragma unroll
    for (int j = 0; j < N; ++j) x[j] += y[j];
  }
}

// q.k of the staged tokens, after a barrier: as many lanes per token as share a column.
template <int D, int P> __device__ __forceinline__ void chain_qk(ChainBlock<D, P>& s) {
  using Cfg = ChainCfg<D, P>;
  const int tid = threadIdx.x, l = tid % Cfg::kLanes;
#pragma unroll
  for (int t0 = 0; t0 < kBlock; t0 += Cfg::kThreads / Cfg::kLanes) {
    const int t = t0 + tid / Cfg::kLanes;
    float d[1] = {0.f};
#pragma unroll
    for (int i = 0; i < Cfg::kRows; i += 4) {
      const float4 x = *reinterpret_cast<const float4*>(&s.q[t][l * Cfg::kLd + i]), y = *reinterpret_cast<const float4*>(&s.k[t][l * Cfg::kLd + i]);
      d[0] += x.x * y.x + x.y * y.y + x.z * y.z + x.w * y.w;
    }
    lanes_sum<D>(d);
    if (l == 0) s.qk[t] = d[0];
  }
}

// A lane's part of a staged row.
template <int D> struct ChainRow {
  static constexpr int kPairs = ChainCfg<D, 1>::kRows / 2;
  float2 x[kPairs];
  __device__ __forceinline__ void load(const float* row) {
#pragma unroll
    for (int i = 0; i < kPairs; i += 2) {
      const float4 r = *reinterpret_cast<const float4*>(row + 2 * i);
      x[i] = f2(r.x, r.y);
      x[i + 1] = f2(r.z, r.w);
    }
  }
  __device__ __forceinline__ float dot(const float2 (&s)[kPairs]) const {
    float2 a = mul2(x[0], s[0]), b = mul2(x[1], s[1]);
#pragma unroll
    for (int i = 2; i < kPairs; i += 2) {
      a = fma2(x[i], s[i], a);
      b = fma2(x[i + 1], s[i + 1], b);
    }
    a = add2(a, b);
    return a.x + a.y;
  }
};

struct ChainParams {
  Params p;
  void* o;           // forward
  float* ST;
  float* e;          // [tokens][H][D]: left by the forward for a backward, or NULL
  float* h;          // [chunks][H][D][D] states at the chunks' starts, or NULL
  const void* d_o;   // reverse
  const float* dST;
  float *y, *dh, *dS0;
  void* dv;
};

// P neighbouring values.
template <int P> struct Columns;
template <> struct Columns<1> { using F = float; };
template <> struct Columns<2> { using F = float2; };
template <> struct Columns<4> { using F = float4; };
template <int P> __device__ __forceinline__ void load_columns(const float* at, float (&x)[P]) {
  const typename Columns<P>::F r = *reinterpret_cast<const typename Columns<P>::F*>(at);
  const float* v = reinterpret_cast<const float*>(&r);
#pragma unroll
  for (int j = 0; j < P; ++j) x[j] = v[j];
}
template <int P> __device__ __forceinline__ void store_columns(float* at, const float (&x)[P]) {
  typename Columns<P>::F r;
#pragma unroll
  for (int j = 0; j < P; ++j) reinterpret_cast<float*>(&r)[j] = x[j];
  *reinterpret_cast<typename Columns<P>::F*>(at) = r;
}
__device__ __forceinline__ void store_columns(bf16* at, const float (&x)[1]) { *at = __float2bfloat16(x[0]); }
__device__ __forceinline__ void store_columns(bf16* at, const float (&x)[2]) {
  *reinterpret_cast<uint32_t*>(at) = pack_bf16(x[0], x[1]);
}
__device__ __forceinline__ void store_columns(bf16* at, const float (&x)[4]) {
  *reinterpret_cast<uint2*>(at) = make_uint2(pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3]));
}

// A lane's rows of its P columns, from and to a state: `at` is its first element.
template <int D, int P> __device__ __forceinline__ void chain_state_in(float2 (&S)[P][ChainRow<D>::kPairs], const float* at) {
#pragma unroll
  for (int i = 0; i < ChainRow<D>::kPairs; ++i) {
    float x[P] = {}, y[P] = {};
    if (at) {
      load_columns(at + (size_t)(2 * i) * D, x);
      load_columns(at + (size_t)(2 * i + 1) * D, y);
    }
#pragma unroll
    for (int j = 0; j < P; ++j) S[j][i] = f2(x[j], y[j]);
  }
}
template <int D, int P> __device__ __forceinline__ void chain_state_out(const float2 (&S)[P][ChainRow<D>::kPairs], float* at) {
#pragma unroll
  for (int i = 0; i < ChainRow<D>::kPairs; ++i) {
    float x[P], y[P];
#pragma unroll
    for (int j = 0; j < P; ++j) {
      x[j] = S[j][i].x;
      y[j] = S[j][i].y;
    }
    store_columns(at + (size_t)(2 * i) * D, x);
    store_columns(at + (size_t)(2 * i + 1) * D, y);
  }
}

template <int D, int P, typename T>
__global__ void __launch_bounds__(ChainCfg<D, P>::kThreads) gdr_chain_fwd_kernel(const ChainParams c) {
  wait_prerequisites();
  using Cfg = ChainCfg<D, P>;
  __shared__ __align__(16) ChainBlock<D, P> s;
  const Params& p = c.p;
  const int H = p.geo.heads, unit = blockIdx.x / Cfg::kGroups, col0 = (blockIdx.x % Cfg::kGroups) * Cfg::kCols;
  const int n = unit / H, h = unit - n * H, hk = h / p.group;
  SeqInfo sq = sequence(p.geo, n);
  const int tid = threadIdx.x, col = tid / Cfg::kLanes * P, lane = tid % Cfg::kLanes;
  const bool mine = col < Cfg::kCols;  // (eight columns leave half a warp idle)
  const size_t sbase = (size_t)unit * D * D + (size_t)lane * Cfg::kRows * D + col0 + (mine ? col : 0);
  constexpr int kPairs = Cfg::kRows / 2;
  float2 S[P][kPairs];  // rows 2 i and 2 i + 1
  chain_state_in<D, P>(S, p.S0 ? p.S0 + sbase : nullptr);
  ChainLoad<D, P, T> next;
  next.fetch(p, p.v, sq, 0, h, hk, col0);
  if (cut_sequence<Cfg::kThreads>(p.geo, n, sq)) next.fetch(p, p.v, sq, 0, h, hk, col0);
  for (int t0 = 0; t0 < sq.len; t0 += kBlock) {
    __syncthreads();
    next.store(s);
    if (t0 + kBlock < sq.len) next.fetch(p, p.v, sq, t0 + kBlock, h, hk, col0);
    if (c.h && t0 % kChunk == 0 && mine) {
      chain_state_out<D, P>(S, c.h + ((size_t)(sq.chunk0 + t0 / kChunk) * H + h) * D * D + (size_t)lane * Cfg::kRows * D + col0 + col);
    }
    __syncthreads();
    chain_qk<D, P>(s);
    ChainRow<D> k, q;
    k.load(&s.k[0][lane * Cfg::kLd]);
    q.load(&s.q[0][lane * Cfg::kLd]);
    __syncthreads();
    const int steps = min(kBlock, sq.len - t0);
#pragma unroll 4
    for (int t = 0; t < steps; ++t) {
      ChainRow<D> kn, qn;  // the next token's (the last one's again at the end of a block)
      const int tn = min(t + 1, kBlock - 1);
      kn.load(&s.k[tn][lane * Cfg::kLd]);
      qn.load(&s.q[tn][lane * Cfg::kLd]);
      const float a = s.a[t], b = s.beta[t], qk = s.qk[t];
      float e[P], o[P], sums[2 * P];  // S^T k, then S^T q
#pragma unroll
      for (int j = 0; j < P; ++j) {
        sums[j] = k.dot(S[j]);
        sums[P + j] = q.dot(S[j]);
      }
      lanes_sum<D>(sums);
#pragma unroll
      for (int j = 0; j < P; ++j) {
        e[j] = s.val[t][mine ? col + j : 0] - a * sums[j];
        const float u = b * e[j];
#pragma unroll
        for (int i = 0; i < kPairs; ++i) S[j][i] = fma2(k.x[i], f2(u, u), mul2(f2(a, a), S[j][i]));
        o[j] = p.scale * (a * sums[P + j] + qk * u);
      }
      if (mine && lane == 0) {
        const size_t at = ((size_t)(sq.bos + t0 + t) * H + h) * D + col0 + col;
        store_columns(static_cast<T*>(c.o) + at, o);
        if (c.e) store_columns(c.e + at, e);
      }
      k = kn;
      q = qn;
    }
  }
  if (c.ST && mine) chain_state_out<D, P>(S, c.ST + sbase);
}

template <int D, int P, typename T>
__global__ void __launch_bounds__(ChainCfg<D, P>::kThreads) gdr_chain_bwd_kernel(const ChainParams c) {
  wait_prerequisites();
  using Cfg = ChainCfg<D, P>;
  __shared__ __align__(16) ChainBlock<D, P> s;
  const Params& p = c.p;
  const int H = p.geo.heads, unit = blockIdx.x / Cfg::kGroups, col0 = (blockIdx.x % Cfg::kGroups) * Cfg::kCols;
  const int n = unit / H, h = unit - n * H, hk = h / p.group;
  const SeqInfo sq = sequence(p.geo, n);
  const int tid = threadIdx.x, col = tid / Cfg::kLanes * P, lane = tid % Cfg::kLanes;
  const bool mine = col < Cfg::kCols;
  const size_t sbase = (size_t)unit * D * D + (size_t)lane * Cfg::kRows * D + col0 + (mine ? col : 0);
  constexpr int kPairs = Cfg::kRows / 2;
  float2 S[P][kPairs];  // dS
  chain_state_in<D, P>(S, c.dST ? c.dST + sbase : nullptr);
  const int last = sq.len > 0 ? (sq.len - 1) / kBlock * kBlock : -kBlock;
  ChainLoad<D, P, T> next;
  if (last >= 0) next.fetch(p, c.d_o, sq, last, h, hk, col0);
  for (int t0 = last; t0 >= 0; t0 -= kBlock) {
    __syncthreads();
    next.store(s);
    if (t0 > 0) next.fetch(p, c.d_o, sq, t0 - kBlock, h, hk, col0);
    if (mine && (t0 == last || (t0 + kBlock) % kChunk == 0)) {  // the state's cotangent at the end of this block's chunk
      chain_state_out<D, P>(S, c.dh + ((size_t)(sq.chunk0 + t0 / kChunk) * H + h) * D * D + (size_t)lane * Cfg::kRows * D + col0 + col);
    }
    __syncthreads();
    chain_qk<D, P>(s);
    const int top = min(kBlock, sq.len - t0) - 1;
    ChainRow<D> k, q;
    k.load(&s.k[top][lane * Cfg::kLd]);
    q.load(&s.q[top][lane * Cfg::kLd]);
    __syncthreads();
#pragma unroll 4
    for (int t = top; t >= 0; --t) {
      ChainRow<D> kn, qn;
      const int tn = max(t - 1, 0);
      kn.load(&s.k[tn][lane * Cfg::kLd]);
      qn.load(&s.q[tn][lane * Cfg::kLd]);
      const float a = s.a[t], b = s.beta[t], qk = s.qk[t];
      float x[P], y[P];
#pragma unroll
      for (int j = 0; j < P; ++j) y[j] = k.dot(S[j]);
      lanes_sum<D>(y);
#pragma unroll
      for (int j = 0; j < P; ++j) {
        const float w = p.scale * s.val[t][mine ? col + j : 0];
        y[j] += qk * w;
        x[j] = b * y[j];
#pragma unroll
        for (int i = 0; i < kPairs; ++i) S[j][i] = mul2(f2(a, a), fma2(k.x[i], f2(-x[j], -x[j]), fma2(q.x[i], f2(w, w), S[j][i])));
      }
      if (mine && lane == 0) {
        const size_t at = ((size_t)(sq.bos + t0 + t) * H + h) * D + col0 + col;
        store_columns(c.y + at, y);
        store_columns(static_cast<T*>(c.dv) + at, x);
      }
      k = kn;
      q = qn;
    }
  }
  if (c.dS0 && mine) chain_state_out<D, P>(S, c.dS0 + sbase);
}

// ------------------------------------------------------------------------------- gradients of a chunk, fp32
struct ChunkGradParams {
  Params p;
  const void* d_o;
  const float *e, *y, *h, *dh;
  void *dq, *dk, *dbeta;
  float* dg;
};

template <int D> struct GradCfg {
  static constexpr int kThreads = 256;
  static constexpr int kLd = D + 4;               // row stride of the [64][D] tiles
  static constexpr int kLdP = 68;                 // row stride of the [64][64] pair matrices
  static constexpr int kTile = kChunk * kLd;
  static constexpr int kSlice = D < 32 ? D : 32;  // state rows staged at a time
  static constexpr int kCols = D / 16 > 0 ? D / 16 : 1;  // channels of a thread (every 16th)
  // q, k, do, e, y, two pair matrices, a slice of a state, scalars
  static constexpr int kStaged = kSlice * kLd > 16 * kChunk ? kSlice * kLd : 16 * kChunk;  // (the column sums pass through it too)
  static constexpr int kFloats = 5 * kTile + 2 * kChunk * kLdP + kStaged + 6 * kChunk;
  static constexpr int kSmem = kFloats * 4;
};

// One CTA per (chunk, key head): the value heads of the group one after the other, their dq and dk added up in registers.
// A thread owns four rows (tokens) and, of the products, four columns or every sixteenth channel.
template <int D, typename T>
__global__ void __launch_bounds__(256) gdr_chunk_grad_kernel(const ChunkGradParams c) {
  wait_prerequisites();
  using Cfg = GradCfg<D>;
  extern __shared__ __align__(16) float smem_f[];
  float* sQ = smem_f;
  float* sK = sQ + Cfg::kTile;
  float* sO = sK + Cfg::kTile;
  float* sE = sO + Cfg::kTile;
  float* sY = sE + Cfg::kTile;
  float* sCq = sY + Cfg::kTile;
  float* sCm = sCq + kChunk * Cfg::kLdP;
  float* sS = sCm + kChunk * Cfg::kLdP;
  float* sG = sS + Cfg::kStaged;
  float* sGl = sG + kChunk;
  float* sB = sGl + kChunk;
  float* sdG = sB + kChunk;       // [64]
  float* sState = sdG + kChunk;   // [64] k.(dS' e) parts
  float* sRed = sState + kChunk;  // scratch [64]
  const Params& p = c.p;
  int n, tok0, valid;
  if (!chunk_lookup(p.geo, blockIdx.x, n, tok0, valid)) return;
  const int H = p.geo.heads, hk = blockIdx.y, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int ti = tid >> 4, tj = tid & 15;
  constexpr int kC = Cfg::kCols;
  const bool chan = tj < D;  // (eight channels leave half the threads without one)

  for (int at = tid; at < kChunk * D; at += 256) {
    const int t = at / D, d = at - t * D;
    float q = 0.f, k = 0.f;
    if (t < valid) {
      const size_t src = ((size_t)(tok0 + t) * p.key_heads + hk) * D + d;
      q = to_f(static_cast<const T*>(p.q)[src]);
      k = to_f(static_cast<const T*>(p.k)[src]);
    }
    sQ[t * Cfg::kLd + d] = q;
    sK[t * Cfg::kLd + d] = k;
  }
  float dq[4][kC], dk[4][kC];
#pragma unroll
  for (int r = 0; r < 4; ++r)
#pragma unroll
    for (int j = 0; j < kC; ++j) dq[r][j] = dk[r][j] = 0.f;

  for (int g = 0; g < p.group; ++g) {
    const int h = hk * p.group + g;
    const size_t sc0 = (size_t)tok0 * H + h;
    __syncthreads();
    for (int at = tid; at < kChunk * D; at += 256) {
      const int t = at / D, d = at - t * D;
      float o = 0.f, e = 0.f, y = 0.f;
      if (t < valid) {
        const size_t src = ((size_t)(tok0 + t) * H + h) * D + d;
        o = to_f(static_cast<const T*>(c.d_o)[src]);
        e = c.e[src];
        y = c.y[src];
      }
      sO[t * Cfg::kLd + d] = o;
      sE[t * Cfg::kLd + d] = e;
      sY[t * Cfg::kLd + d] = y;
    }
    if (warp == 0) chunk_scalars<T>(p, sc0, valid, sG, sGl, sB);
    if (tid < kChunk) sdG[tid] = 0.f;
    __syncthreads();
    const float GL = sG[kChunk - 1], GLl = sGl[kChunk - 1];

    // ---- pair matrices: rows 4 ti .. 4 ti + 3, columns tj + 16 j
    {
      float f1[4][4], f2[4][4], qk[4][4], kk[4][4];
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int j = 0; j < 4; ++j) f1[r][j] = f2[r][j] = qk[r][j] = kk[r][j] = 0.f;
#pragma unroll 2
      for (int d = 0; d < D; ++d) {
        float ro[4], ry[4], rq[4], rk[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int at = (4 * ti + r) * Cfg::kLd + d;
          ro[r] = sO[at]; ry[r] = sY[at]; rq[r] = sQ[at]; rk[r] = sK[at];
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int at = (tj + 16 * j) * Cfg::kLd + d;
          const float ce = sE[at], ck = sK[at];
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            f1[r][j] += ro[r] * ce; f2[r][j] += ry[r] * ce; qk[r][j] += rq[r] * ck; kk[r][j] += rk[r] * ck;
          }
        }
      }
      float rows[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int jj = tj + 16 * j;
        float column = 0.f;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int i = 4 * ti + r;
          const float decay = i >= jj ? decay_between(sG[i], sGl[i], sG[jj], sGl[jj]) : 0.f;
          const float cq = i >= jj ? p.scale * sB[jj] * decay * f1[r][j] : 0.f;
          const float cm = i > jj ? -sB[i] * sB[jj] * decay * f2[r][j] : 0.f;
          sCq[i * Cfg::kLdP + jj] = cq;
          sCm[i * Cfg::kLdP + jj] = cm;
          if (i == jj && i < valid) store_dbeta<T>(p, c.dbeta, sc0 + (size_t)i * H, f2[r][j]);
          const float x = i == jj ? 0.f : cq * qk[r][j] + cm * kk[r][j];  // (a pair of a token with itself moves no gate)
          rows[r] += x;
          column += x;
        }
        // the column's sum over the sixteen row groups, in a fixed order below
        sS[ti * kChunk + jj] = column;
      }
#pragma unroll
      for (int r = 0; r < 4; ++r) {
#pragma unroll
        for (int o = 8; o; o >>= 1) rows[r] += __shfl_xor_sync(0xffffffffu, rows[r], o);
        if (tj == 0) sRed[4 * ti + r] = rows[r];
      }
    }
    __syncthreads();
    if (tid < kChunk) {
      float x = sRed[tid];
#pragma unroll
      for (int w = 0; w < 16; ++w) x -= sS[w * kChunk + tid];
      sdG[tid] = x;
    }

    // ---- the pair parts of dq and dk
    if (chan) {
#pragma unroll 2
      for (int m = 0; m < kChunk; ++m) {
        float cq[4], cm[4], cqt[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int i = 4 * ti + r;
          cq[r] = sCq[i * Cfg::kLdP + m];
          cqt[r] = sCq[m * Cfg::kLdP + i];
          cm[r] = sCm[i * Cfg::kLdP + m] + sCm[m * Cfg::kLdP + i];
        }
#pragma unroll
        for (int j = 0; j < kC; ++j) {
          const int d = tj + 16 * j;
          const float kv = sK[m * Cfg::kLd + d], qv = sQ[m * Cfg::kLd + d];
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            dq[r][j] += cq[r] * kv;
            dk[r][j] += cqt[r] * qv + cm[r] * kv;
          }
        }
      }
    }

    // ---- the state parts: channels kSlice at a time (thread: 4 tokens, channel tj (+ 16) of the slice)
    float inter[4] = {0.f, 0.f, 0.f, 0.f}, carry[4] = {0.f, 0.f, 0.f, 0.f}, dot = 0.f;
    const float* hs = c.h + ((size_t)blockIdx.x * H + h) * D * D;
    const float* ds = c.dh + ((size_t)blockIdx.x * H + h) * D * D;
#pragma unroll
    for (int part = 0; part < D / Cfg::kSlice; ++part) {
      for (int which = 0; which < 2; ++which) {
        const float* src = (which ? ds : hs) + (size_t)part * Cfg::kSlice * D;
        __syncthreads();
        for (int at = tid; at < Cfg::kSlice * D; at += 256) {
          const float x = src[at];
          if (which) dot += x * hs[(size_t)part * Cfg::kSlice * D + at];
          sS[at / D * Cfg::kLd + at % D] = x;
        }
        __syncthreads();
#pragma unroll
        for (int jj = 0; jj < (Cfg::kSlice + 15) / 16; ++jj) {
          const int local = tj + 16 * jj, d = part * Cfg::kSlice + local;
          if (local >= Cfg::kSlice) continue;
          const int j = part * ((Cfg::kSlice + 15) / 16) + jj;  // channel d = tj + 16 j
          float a0[4] = {0.f, 0.f, 0.f, 0.f}, a1[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
          for (int v = 0; v < D; ++v) {
            const float x = sS[local * Cfg::kLd + v];
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              const int at = (4 * ti + r) * Cfg::kLd + v;
              if (which) {
                a0[r] += x * sE[at];
              } else {
                a0[r] += x * sO[at];
                a1[r] += x * sY[at];
              }
            }
          }
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int i = 4 * ti + r;
            const float kv = sK[i * Cfg::kLd + d];
            if (which) {
              const float x = decay_between(GL, GLl, sG[i], sGl[i]) * sB[i] * a0[r];
              dk[r][j] += x;
              carry[r] += kv * x;
            } else {
              const float gam = decay_between(sG[i], sGl[i], 0.f, 0.f), x = p.scale * gam * a0[r], w = -gam * sB[i] * a1[r];
              dq[r][j] += x;
              dk[r][j] += w;
              inter[r] += sQ[i * Cfg::kLd + d] * x + kv * w;
            }
          }
        }
      }
    }
    // ---- dG: what the states carry in is the token's own, what they carry out goes to the chunk's last token as well
#pragma unroll
    for (int r = 0; r < 4; ++r) {
#pragma unroll
      for (int o = 8; o; o >>= 1) {
        inter[r] += __shfl_xor_sync(0xffffffffu, inter[r], o);
        carry[r] += __shfl_xor_sync(0xffffffffu, carry[r], o);
      }
      if (tj == 0) {
        sState[4 * ti + r] = carry[r];
        sRed[4 * ti + r] = inter[r] - carry[r];
      }
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, o);
    __syncthreads();
    if (lane == 0) sS[warp] = dot;
    __syncthreads();
    if (warp == 0) {  // reverse cumulative sum: lane l has tokens 2 l and 2 l + 1
      float whole = 0.f;
#pragma unroll
      for (int w = 0; w < 8; ++w) whole += sS[w];
      float out = sState[2 * lane] + sState[2 * lane + 1];
#pragma unroll
      for (int o = 16; o; o >>= 1) out += __shfl_xor_sync(0xffffffffu, out, o);
      const float end = out + decay_between(GL, GLl, 0.f, 0.f) * whole;
      float x0 = sdG[2 * lane] + sRed[2 * lane], x1 = sdG[2 * lane + 1] + sRed[2 * lane + 1];
      float run = x0 + x1;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const float z = __shfl_down_sync(0xffffffffu, run, o);
        if (lane + o < 32) run += z;
      }
      if (2 * lane < valid) c.dg[sc0 + (size_t)(2 * lane) * H] = run + end;
      if (2 * lane + 1 < valid) c.dg[sc0 + (size_t)(2 * lane + 1) * H] = run - x0 + end;
    }
  }
  if (chan) {
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int t = 4 * ti + r;
      if (t >= valid) continue;
#pragma unroll
      for (int j = 0; j < kC; ++j) {
        const size_t at = ((size_t)(tok0 + t) * p.key_heads + hk) * D + tj + 16 * j;
        static_cast<T*>(c.dq)[at] = from_f<T>(dq[r][j]);
        static_cast<T*>(c.dk)[at] = from_f<T>(dk[r][j]);
      }
    }
  }
}

// ------------------------------------------------------------------------------------------------ host side
// Columns of a lane.  A warp reads every key from shared memory for the columns that it has, so with several CTAs on an SM more
// columns a lane are faster, with one CTA each the shorter turn is.  Measured, 512 tokens forward + reverse, by the CTAs that one
// column a lane would make: 128 columns, 256 CTAs 292 / 308 / 422 us with 1 / 2 / 4, 512 CTAs 599 / 434 / 423, 1,024 CTAs
// 969 / 826 / 684; 64 columns, 256 CTAs 218 / 200 / 295, 512 CTAs 322 / 268 / 295, 1,024 CTAs 607 / 490 / 487.
template <int D> static int lane_columns(int units) {
  const long long ctas = (long long)units * ChainCfg<D, 1>::kGroups;
  const int sms = sm_count();
  if (D == 128 && ctas > 3 * sms) return 4;
  return D >= 32 && ctas > 2 * sms ? 2 : 1;
}

template <int D, int P, typename T> static int launch_chain(const ChainParams& c, bool reverse, cudaStream_t st) {
  using Cfg = ChainCfg<D, P>;
  const int ctas = c.p.geo.n_seqs * c.p.geo.heads * Cfg::kGroups;
  return launch_kernel(reverse ? gdr_chain_bwd_kernel<D, P, T> : gdr_chain_fwd_kernel<D, P, T>, ctas, Cfg::kThreads, 0, st, c);
}
template <int D, typename T> static int launch_chain(const ChainParams& c, bool reverse, cudaStream_t st) {
  const int columns = lane_columns<D>(c.p.geo.n_seqs * c.p.geo.heads);
  if constexpr (D == 128)
    if (columns == 4) return launch_chain<D, 4, T>(c, reverse, st);
  if constexpr (D >= 32)
    if (columns == 2) return launch_chain<D, 2, T>(c, reverse, st);
  return launch_chain<D, 1, T>(c, reverse, st);
}

template <int D, typename T> static int launch_recurrent(const ChainParams& c, bool few, cudaStream_t st) {
  const int units = c.p.geo.n_seqs * c.p.geo.heads;
  begin_stage(kStageGdrRecurrent, st);
  int rc;
  if (few) {
    RecurrentParams r;
    r.p = c.p; r.o = c.o; r.ST = c.ST;
    rc = launch_kernel(gdr_few_kernel<D, T>, units, FewCfg<D>::kThreads, 0, st, r);
  } else {
    rc = launch_chain<D, T>(c, false, st);
  }
  end_stage(st);
  return rc;
}

template <int D, typename T> static int launch_reverse(const ChainParams& c, const ChunkGradParams& g, cudaStream_t st) {
  begin_stage(kStageGdrRecurrentBwd, st);
  int rc = launch_chain<D, T>(c, true, st);
  end_stage(st);
  if (rc != PKDA_OK) return rc;
  if (!ensure_dynamic_smem(gdr_chunk_grad_kernel<D, T>, GradCfg<D>::kSmem)) return PKDA_ERR_LAUNCH;
  begin_stage(kStageGdrChunkGrad, st);
  rc = launch_kernel(gdr_chunk_grad_kernel<D, T>, dim3(c.p.geo.total_chunks, c.p.key_heads), 256, GradCfg<D>::kSmem, st, g);
  end_stage(st);
  return rc;
}

template <typename F> static int by_width(int D, F&& f) {
  switch (D) {
    case 8: return f(std::integral_constant<int, 8>());
    case 16: return f(std::integral_constant<int, 16>());
    case 32: return f(std::integral_constant<int, 32>());
    case 64: return f(std::integral_constant<int, 64>());
    case 128: return f(std::integral_constant<int, 128>());
    default: return PKDA_ERR_SHAPE;
  }
}

// Rows of one or two tokens keep the whole state in one CTA's registers; longer ones split its columns.
static bool few_tokens(const pkda_gdr_problem& p) { return !p.cu_seqlens && p.seq_len <= 2; }

int exact_forward(const pkda_gdr_problem& p, const Params& base, void* o, float* final_state, float* e, float* h, cudaStream_t st) {
  ChainParams c = {};
  c.p = base; c.o = o; c.ST = final_state; c.e = e; c.h = h;
  const bool few = few_tokens(p) && !e;
  return by_width(p.head_dim, [&](auto d) {
    constexpr int D = decltype(d)::value;
    return act_dtype(p) == PKDA_BF16 ? launch_recurrent<D, bf16>(c, few, st) : launch_recurrent<D, float>(c, few, st);
  });
}

int exact_backward(const pkda_gdr_problem& p, const Params& base, const pkda_gdr_bwd_args& a, const float* e, const float* h, float* y,
                   float* dh, cudaStream_t st) {
  ChainParams c = {};
  c.p = base; c.d_o = a.d_o; c.dST = a.d_final_state; c.y = y; c.dh = dh; c.dS0 = a.d_initial_state; c.dv = a.dv;
  ChunkGradParams g = {};
  g.p = base; g.d_o = a.d_o; g.e = e; g.y = y; g.h = h; g.dh = dh; g.dq = a.dq; g.dk = a.dk; g.dbeta = a.dbeta; g.dg = a.dg;
  return by_width(p.head_dim, [&](auto d) {
    constexpr int D = decltype(d)::value;
    return act_dtype(p) == PKDA_BF16 ? launch_reverse<D, bf16>(c, g, st) : launch_reverse<D, float>(c, g, st);
  });
}

}  // namespace gdr
}  // namespace pkda
