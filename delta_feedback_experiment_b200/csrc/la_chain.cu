// Linear attention token by token, in fp32: the decoding step, short prompts, and the forward and backward of fp32 activations and of
// the head widths that the chunked kernels do not take.
//
// A CTA takes some of the value columns of one (sequence, head).  A thread holds four columns of some rows of the state, a warp reads
// whole rows of it; per token it decays them, takes the product with x, adds y z^T.  The products are summed over the threads of a
// column by shuffles inside a warp and through shared memory across them, several tokens at a time, since no token waits for the
// sums.  The token's own write is left out of them and added by the scalar x.y, so that the gate's gradient sees the reads of the
// other tokens alone (la_common.cuh).
#include "la_common.cuh"

namespace pkda {
namespace la {

template <int D, int kCols> struct ChainCfg {
  static constexpr int kLanes = kCols / 4;                                       // threads of a row
  static constexpr int kGroups = 256 / kLanes < D / 4 ? 256 / kLanes : (D >= 4 ? D / 4 : 1);  // row groups
  static constexpr int kRows = D / kGroups;                                      // rows of a thread
  static constexpr int kActive = kLanes * kGroups;
  static constexpr int kThreads = kActive < 32 ? 32 : kActive;
  static constexpr int kWarps = kThreads / 32;
  static constexpr int kBlock = kCols >= 128 ? 4 : kCols >= 64 ? 8 : 16;         // tokens of a block
};

__device__ __forceinline__ float4 read4(const bf16* p) {
  const uint2 r = *reinterpret_cast<const uint2*>(p);
  const float2 a = unpack_bf16(r.x), b = unpack_bf16(r.y);
  return make_float4(a.x, a.y, b.x, b.y);
}
__device__ __forceinline__ float4 read4(const float* p) { return *reinterpret_cast<const float4*>(p); }

struct ChainParams {
  Call c;
  Pass pass[3];
};

template <int D, int kCols, typename T>
__global__ void __launch_bounds__(ChainCfg<D, kCols>::kThreads, D * kCols >= 128 * 128 ? 2 : 1) la_chain_kernel(const __grid_constant__ ChainParams a) {
  after_previous();
  using Cfg = ChainCfg<D, kCols>;
  constexpr int kBlock = Cfg::kBlock, kRows = Cfg::kRows, kThreads = Cfg::kThreads, kWarps = Cfg::kWarps, kLanes = Cfg::kLanes;
  constexpr int kSlices = D / kCols;
  const Pass& p = a.pass[blockIdx.y];
  const Geo& geo = a.c.geo;
  const int H = geo.heads, unit = blockIdx.x / kSlices, slice = blockIdx.x - unit * kSlices, n = unit / H, h = unit - n * H;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, col0 = slice * kCols;
  const int kg = tid / kLanes, cq = tid - kg * kLanes, row0 = kg * kRows;
  const bool active = tid < Cfg::kActive, rev = p.reverse;
  __shared__ __align__(16) float s_x[kBlock][D], s_y[kBlock][D], s_z[kBlock][kCols], s_u[kBlock][kCols];
  __shared__ __align__(16) float s_part[kBlock][kWarps][kCols];
  __shared__ float s_a[kBlock], s_d[kBlock], s_dot[kBlock][(kCols + 31) / 32];

  float4 S[kRows];  // rows row0.., columns col0 + 4 cq..
  const size_t sbase = (size_t)unit * D * D;
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    S[i] = make_float4(0.f, 0.f, 0.f, 0.f);
    if (p.init && active) {
      if (!p.init_t) {
        S[i] = *reinterpret_cast<const float4*>(p.init + sbase + (size_t)(row0 + i) * D + col0 + 4 * cq);
      } else {
        const float* at = p.init + sbase + (size_t)(col0 + 4 * cq) * D + row0 + i;
        S[i] = make_float4(at[0], at[D], at[2 * D], at[3 * D]);
      }
    }
  }
  SeqInfo sq = gdr::sequence(geo, n);
  gdr::cut_sequence<kThreads>(geo, n, sq);
  const size_t xs = (size_t)(H / p.x_group) * D, ys = (size_t)(H / p.y_group) * D, zs = (size_t)(H / p.z_group) * D;
  const T* x = static_cast<const T*>(p.x) + (size_t)(h / p.x_group) * D;
  const T* y = static_cast<const T*>(p.y) + (size_t)(h / p.y_group) * D;
  const T* z = static_cast<const T*>(p.z) + (size_t)(h / p.z_group) * D + col0;
  const size_t us = p.u ? (size_t)(H / p.u_group) * D : 0;
  const T* u = p.u ? static_cast<const T*>(p.u) + (size_t)(h / p.u_group) * D + col0 : nullptr;

  for (int t0 = 0; t0 < sq.len; t0 += kBlock) {
    const int count = min(kBlock, sq.len - t0);
    auto token = [&](int t) { return (size_t)(sq.bos + (rev ? sq.len - 1 - t0 - t : t0 + t)); };
    for (int i = tid; i < count * (D / 4); i += kThreads) {
      const int t = i / (D / 4), c = 4 * (i - t * (D / 4));
      const size_t tok = token(t);
      *reinterpret_cast<float4*>(&s_x[t][c]) = read4(x + tok * xs + c);
      *reinterpret_cast<float4*>(&s_y[t][c]) = read4(y + tok * ys + c);
    }
    for (int i = tid; i < count * kLanes; i += kThreads) {
      const int t = i / kLanes, c = 4 * (i - t * kLanes);
      const size_t tok = token(t);
      *reinterpret_cast<float4*>(&s_z[t][c]) = read4(z + tok * zs + c);
      if (u) *reinterpret_cast<float4*>(&s_u[t][c]) = read4(u + tok * us + c);
    }
    if (tid < count) s_a[tid] = expf(gate(a.c, token(tid), h));
    __syncthreads();
    for (int t = warp; t < count; t += kWarps) {  // x.y
      float d = 0.f;
      for (int c = lane; c < D; c += 32) d = fmaf(s_x[t][c], s_y[t][c], d);
#pragma unroll
      for (int o = 16; o; o >>= 1) d += __shfl_xor_sync(0xffffffffu, d, o);
      if (lane == 0) s_d[t] = d;
    }
    for (int t = 0; t < count; ++t) {
      const float dec = s_a[t];
      float2 acc[2] = {f2(0.f, 0.f), f2(0.f, 0.f)};
      if (active) {
        const float4 zv = *reinterpret_cast<const float4*>(&s_z[t][4 * cq]);
        const float2 z0 = f2(p.write * zv.x, p.write * zv.y), z1 = f2(p.write * zv.z, p.write * zv.w), dd = f2(dec, dec);
#pragma unroll
        for (int i = 0; i < kRows; ++i) {
          const float xv = s_x[t][row0 + i], yv = s_y[t][row0 + i];
          float2 lo = f2(S[i].x, S[i].y), hi = f2(S[i].z, S[i].w);
          if (!rev) {
            lo = mul2(lo, dd);
            hi = mul2(hi, dd);
          }
          acc[0] = fma2(lo, f2(xv, xv), acc[0]);
          acc[1] = fma2(hi, f2(xv, xv), acc[1]);
          lo = fma2(f2(yv, yv), z0, lo);
          hi = fma2(f2(yv, yv), z1, hi);
          if (rev) {
            lo = mul2(lo, dd);
            hi = mul2(hi, dd);
          }
          S[i] = make_float4(lo.x, lo.y, hi.x, hi.y);
        }
      }
#pragma unroll
      for (int o = 16; o >= kLanes; o >>= 1) {
        acc[0].x += __shfl_xor_sync(0xffffffffu, acc[0].x, o);
        acc[0].y += __shfl_xor_sync(0xffffffffu, acc[0].y, o);
        acc[1].x += __shfl_xor_sync(0xffffffffu, acc[1].x, o);
        acc[1].y += __shfl_xor_sync(0xffffffffu, acc[1].y, o);
      }
      if (lane < kLanes) *reinterpret_cast<float4*>(&s_part[t][warp][4 * cq]) = make_float4(acc[0].x, acc[0].y, acc[1].x, acc[1].y);
    }
    __syncthreads();
    // (whole warps: a block has a multiple of 32 columns)
    for (int i = tid; i < kBlock * kCols; i += kThreads) {
      const int t = i / kCols, c = i - t * kCols;
      float dot = 0.f;
      if (t < count) {
        float pre = 0.f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) pre += s_part[t][w][c];
        pre *= p.read;
        const size_t at = (token(t) * H + h) * D + col0 + c;
        if (p.out) {
          const float o = fmaf(p.c * s_d[t], s_z[t][c], pre);
          if (p.out32) static_cast<float*>(p.out)[at] = o;
          else static_cast<T*>(p.out)[at] = from_f<T>(o);
        }
        if (u) dot = pre * s_u[t][c];
      }
      if (p.dots) {
        constexpr int kWidth = kCols < 32 ? kCols : 32;
#pragma unroll
        for (int o = kWidth / 2; o; o >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, o);
        if (c % kWidth == 0) s_dot[t][c / 32] = dot;
      }
    }
    __syncthreads();
    if (p.dots && tid < count) {
      float dot = 0.f;
#pragma unroll
      for (int i = 0; i < (kCols + 31) / 32; ++i) dot += s_dot[tid][i];
      p.dots[((size_t)slice * geo.total_tokens + token(tid)) * H + h] = dot;
    }
  }
  if (active) {
    for (float* fin : {p.fin, p.fin2}) {
      if (!fin) continue;
#pragma unroll
      for (int i = 0; i < kRows; ++i) {
        if (!p.fin_t) {
          *reinterpret_cast<float4*>(fin + sbase + (size_t)(row0 + i) * D + col0 + 4 * cq) = S[i];
        } else {
          float* at = fin + sbase + (size_t)(col0 + 4 * cq) * D + row0 + i;
          at[0] = S[i].x; at[D] = S[i].y; at[2 * D] = S[i].z; at[3 * D] = S[i].w;
        }
      }
    }
  }
}

// Columns of a CTA: as many as leave a CTA for every SM, 16 at least.
static int chain_cols(long long units, int D) {
  int cols = D;
  while (cols > 16 && units * (D / cols) < sm_count()) cols /= 2;
  return cols;
}
int chain_slices(long long units, int D) { return D / chain_cols(units, D); }

template <int D, int kCols, typename T> static int launch(const ChainParams& a, int n, cudaStream_t st) {
  begin_stage(kStageLaChain, st);
  const int rc = launch_kernel(la_chain_kernel<D, kCols, T>, dim3((unsigned)((long long)a.c.geo.n_seqs * a.c.geo.heads * (D / kCols)), n),
                               ChainCfg<D, kCols>::kThreads, 0, st, a);
  end_stage(st);
  return rc;
}
template <int D, typename T> static int launch_cols(const ChainParams& a, int n, int cols, cudaStream_t st) {
  if constexpr (D >= 128)
    if (cols == 128) return launch<D, 128, T>(a, n, st);
  if constexpr (D >= 64)
    if (cols == 64) return launch<D, 64, T>(a, n, st);
  if constexpr (D >= 32)
    if (cols == 32) return launch<D, 32, T>(a, n, st);
  return launch<D, D < 16 ? D : 16, T>(a, n, st);
}
template <typename T> static int launch_width(const ChainParams& a, int D, int n, int cols, cudaStream_t st) {
  switch (D) {
    case 8: return launch_cols<8, T>(a, n, cols, st);
    case 16: return launch_cols<16, T>(a, n, cols, st);
    case 32: return launch_cols<32, T>(a, n, cols, st);
    case 64: return launch_cols<64, T>(a, n, cols, st);
    default: return launch_cols<128, T>(a, n, cols, st);
  }
}
int launch_chain(const Call& c, int D, int dtype, const Pass* passes, int n, cudaStream_t st) {
  ChainParams a;
  a.c = c;
  for (int i = 0; i < n; ++i) a.pass[i] = passes[i];
  const int cols = chain_cols((long long)c.geo.n_seqs * c.geo.heads, D);
  return dtype == PKDA_BF16 ? launch_width<bf16>(a, D, n, cols, st) : launch_width<float>(a, D, n, cols, st);
}

// ------------------------------------------------------------------------------------------------ the gate's gradient
// One CTA per (sequence, head, segment), 256 tokens a turn from the end; sums in 64 bits, since the tokens' shares differ in sign.
__device__ __forceinline__ double warp_suffix(double x, int lane) {  // sum over this lane and those behind it
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const double y = __shfl_down_sync(0xffffffffu, x, o);
    if (lane + o < 32) x += y;
  }
  return x;
}

__global__ void __launch_bounds__(256) la_gate_grad_kernel(const GateGrad a) {
  after_previous();
  const Geo& geo = a.c.geo;
  const int H = geo.heads, unit = blockIdx.x / a.n_items_seq, seg = blockIdx.x - unit * a.n_items_seq, n = unit / H, h = unit - n * H;
  const SeqInfo sq = gdr::sequence(geo, n);
  const int per = a.chunks ? a.chunks * kChunk : max(sq.len, 1), begin = seg * per, end = min(sq.len, begin + per);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  __shared__ double s_sum[8];
  double carry = 0.0, mine = 0.0;
  if (begin < end || seg == 0) {
    if (a.X) {
      carry = a.X[blockIdx.x];
    } else if (a.S && a.dS) {
      const size_t at = (size_t)unit * a.D * a.D;
      double x = 0.0;
      for (int i = tid; i < a.D * a.D; i += 256) x += (double)a.S[at + i] * (double)a.dS[at + i];
#pragma unroll
      for (int o = 16; o; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
      if (lane == 0) s_sum[warp] = x;
      __syncthreads();
      for (int w = 0; w < 8; ++w) carry += s_sum[w];
      __syncthreads();
    }
  }
  for (int last = end; last > begin; last -= 256) {
    const int t = last - 256 + tid;
    const size_t at = (size_t)(sq.bos + t) * H + h;
    double x = 0.0;
    if (t >= begin)
      for (int s = 0; s < a.slices; ++s)
        x += (double)a.row[(size_t)s * geo.total_tokens * H + at] - (double)a.col[(size_t)s * geo.total_tokens * H + at];
    x = warp_suffix(x, lane);
    if (lane == 0) s_sum[warp] = x;
    __syncthreads();
    double all = 0.0;
    for (int w = 0; w < 8; ++w) {
      if (w > warp) x += s_sum[w];
      all += s_sum[w];
    }
    x += carry;
    if (t >= begin) {
      if (a.dg) a.dg[at] = (float)x;
      mine += x;
    }
    carry += all;
    __syncthreads();
  }
  if (a.part) {
    mine = warp_suffix(mine, lane);
    if (lane == 0) s_sum[warp] = mine;
    __syncthreads();
    if (tid == 0) {
      double all = 0.0;
      for (int w = 0; w < 8; ++w) all += s_sum[w];
      a.part[blockIdx.x] = all;
    }
  }
}

// One warp a head: the items' sums in a fixed order.
__global__ void __launch_bounds__(32) la_gate_sum_kernel(const double* part, int n_seqs, int heads, int items, float* dg) {
  after_previous();
  const int h = blockIdx.x, lane = threadIdx.x;
  double x = 0.0;
  for (int i = lane; i < n_seqs * items; i += 32) x += part[((size_t)(i / items) * heads + h) * items + i % items];
#pragma unroll
  for (int o = 16; o; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
  if (lane == 0) dg[h] = (float)x;
}

int launch_gate_grad(const GateGrad& a, cudaStream_t st) {
  begin_stage(kStageLaGate, st);
  int rc = launch_kernel(la_gate_grad_kernel, dim3((unsigned)((long long)a.c.geo.n_seqs * a.c.geo.heads * a.n_items_seq)), 256, 0, st, a);
  end_stage(st);
  if (rc != PKDA_OK || !a.part) return rc;
  begin_stage(kStageLaGate, st);
  rc = launch_kernel(la_gate_sum_kernel, a.c.geo.heads, 32, 0, st, a.part, a.c.geo.n_seqs, a.c.geo.heads, a.n_items_seq, a.dg_head);
  end_stage(st);
  return rc;
}

// ------------------------------------------------------------------------------------------------ shared key heads
template <typename T>
__global__ void __launch_bounds__(256) la_group_sum_kernel(const float4* part, T* out, long long quads, int group, int per_head) {
  after_previous();
  for (long long i = blockIdx.x * 256ll + threadIdx.x; i < quads; i += gridDim.x * 256ll) {
    const long long row = i / per_head;  // (token, key head)
    const float4* at = part + row * group * per_head + (i - row * per_head);
    float4 s = at[0];
    for (int j = 1; j < group; ++j) {
      const float4 x = at[(size_t)j * per_head];
      s.x += x.x; s.y += x.y; s.z += x.z; s.w += x.w;
    }
    if constexpr (sizeof(T) == 4) reinterpret_cast<float4*>(out)[i] = s;
    else reinterpret_cast<uint2*>(out)[i] = make_uint2(pack_bf16(s.x, s.y), pack_bf16(s.z, s.w));
  }
}
int launch_group_sum(const float* part, void* out, int dtype, long long tokens, int key_heads, int group, int D, cudaStream_t st) {
  const long long quads = tokens * key_heads * (D / 4);
  const int grid = (int)(quads < 256ll * 8 * sm_count() ? (quads + 255) / 256 : 8ll * sm_count());
  begin_stage(kStageLaGroup, st);
  const float4* in = reinterpret_cast<const float4*>(part);
  const int rc = dtype == PKDA_BF16 ? launch_kernel(la_group_sum_kernel<bf16>, grid, 256, 0, st, in, static_cast<bf16*>(out), quads, group, D / 4)
                                    : launch_kernel(la_group_sum_kernel<float>, grid, 256, 0, st, in, static_cast<float*>(out), quads, group, D / 4);
  end_stage(st);
  return rc;
}

}  // namespace la
}  // namespace pkda
