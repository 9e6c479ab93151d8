// Linear attention token by token, in fp32: the decoding step, short prompts, and the forward and backward of fp32 activations and of
// the head widths that the chunked kernels do not take.
//
// A CTA takes some of the value columns of one (sequence, head).  A thread holds four columns of some rows of the state, a warp reads
// whole rows of it; per token it decays them, takes the product with x, adds y z^T.  The products are summed over the threads of a
// column by shuffles inside a warp and through shared memory across them, several tokens at a time, since no token waits for the
// sums.  The token's own write is left out of them and added by the scalar x.y, so that the gate's gradient sees the reads of the
// other tokens alone (la_common.cuh).
//
// Bound by the tokens' dependence, 0.5 us each with 128 rows of 128 channels (48 tokens 26 us) and 0.15 us of 64 in fp32 with
// columns spread over SMs, rows a block ahead and four tokens' sums together (2 x 512 tokens of 4 heads, forward and backward, 218 us, 360 without).
//
// For the gate's gradient the forward leaves its state every 256 tokens, and the walk that has its cotangent takes the product of both there.
#include "la_common.cuh"

namespace pkda {
namespace la {

template <int D, int kCols> struct ChainCfg {
  static constexpr int kLanes = kCols / 4;                                       // threads of a row
  static constexpr int kGroups = 256 / kLanes < D / 4 ? 256 / kLanes : (D >= 4 ? D / 4 : 1);  // row groups
  static constexpr int kRows = D / kGroups;                                      // rows of a thread
  static_assert(kRows % 4 == 0, "rows are read four at a time");
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
  ChainEnds e;
  Pass pass[3];
};

// kEnds: with ChainEnds (4 x 48 tokens of 16 heads without: 26.16 us, 26.34 with their tests in the way).
template <int D, int kCols, typename T, bool kEnds>
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
  const bool active = tid < Cfg::kActive, rev = kept(p.reverse) != 0, out32 = kept(p.out32) != 0;
  const float write = kept(p.write), read = kept(p.read), pair_scale = kept(p.c);
  void* const out = kept(static_cast<char*>(p.out));
  float* const dots = kept(p.dots);
  __shared__ __align__(16) float s_x[kBlock][D], s_y[kBlock][D], s_z[kBlock][kCols], s_u[kBlock][kCols];
  __shared__ __align__(16) float s_part[kBlock][kWarps][kCols];
  __shared__ float s_a[kBlock], s_al[kBlock], s_d[kBlock], s_dot[kBlock][(kCols + 31) / 32];

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

  // What a thread has of a block on its way into shared memory: asked for while the block before is worked on.
  constexpr int kX = (kBlock * D / 4 + kThreads - 1) / kThreads, kZ = (kBlock * kLanes + kThreads - 1) / kThreads;
  float4 rx[kX], ry[kX], rz[kZ], ru[kZ];
  float rg = 0.f;
  auto token_of = [&](int at) { return (size_t)(sq.bos + (rev ? sq.len - 1 - at : at)); };
  auto fetch = [&](int t0) {
#pragma unroll
    for (int k = 0; k < kX; ++k) {
      const int i = tid + k * kThreads, t = i / (D / 4), c = 4 * (i % (D / 4));
      if (t < kBlock && t0 + t < sq.len) {
        const size_t tok = token_of(t0 + t);
        rx[k] = read4(x + tok * xs + c);
        ry[k] = read4(y + tok * ys + c);
      }
    }
#pragma unroll
    for (int k = 0; k < kZ; ++k) {
      const int i = tid + k * kThreads, t = i / kLanes, c = 4 * (i % kLanes);
      if (t < kBlock && t0 + t < sq.len) {
        const size_t tok = token_of(t0 + t);
        rz[k] = read4(z + tok * zs + c);
        if (u) ru[k] = read4(u + tok * us + c);
      }
    }
    if (tid < kBlock && t0 + tid < sq.len) rg = gate(a.c, token_of(t0 + tid), h);
  };
  if (sq.len > 0) fetch(0);

  const int span = a.e.segments.chunks * kChunk;
  float* const ends = kEnds ? kept(blockIdx.y == 0 ? a.e.ends : nullptr) : nullptr;
  float* const X = kEnds ? kept(blockIdx.y == gridDim.y - 1 ? a.e.X : nullptr) : nullptr;
  const size_t entry0 = ends || X ? (size_t)first_entry(geo, a.e.segments, n) * H + h : 0;
  const size_t own = (size_t)row0 * D + col0 + 4 * cq;
  int count;
  for (int t0 = 0; t0 < sq.len; t0 += kEnds ? count : kBlock) {
    count = min(kBlock, sq.len - t0);
    if (kEnds && rev && t0 == 0 && sq.len % kBlock) count = sq.len % kBlock;  // (blocks end where segments do: backwards the first one is the short one)
    if (X && (t0 == 0 || (sq.len - t0) % span == 0)) {  // <state, R> at the end of a segment
      const size_t e = entry0 + (size_t)((sq.len - t0 - 1) / span) * H;
      float dot = 0.f;
      if (active) {
        const float* s = a.e.X_states + e * D * D + own;
#pragma unroll
        for (int i = 0; i < kRows; ++i) {
          const float4 v = *reinterpret_cast<const float4*>(s + (size_t)i * D);
          dot = fmaf(v.x, S[i].x, fmaf(v.y, S[i].y, fmaf(v.z, S[i].z, fmaf(v.w, S[i].w, dot))));
        }
      }
#pragma unroll
      for (int o = 16; o; o >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, o);
      if (lane == 0) X[e * (kSlices * kWarps) + slice * kWarps + warp] = dot;
    }
    auto token = [&](int t) { return token_of(t0 + t); };
#pragma unroll
    for (int k = 0; k < kX; ++k) {
      const int i = tid + k * kThreads, t = i / (D / 4), c = 4 * (i % (D / 4));
      if (t < kBlock) {
        *reinterpret_cast<float4*>(&s_x[t][c]) = rx[k];
        *reinterpret_cast<float4*>(&s_y[t][c]) = ry[k];
      }
    }
#pragma unroll
    for (int k = 0; k < kZ; ++k) {
      const int i = tid + k * kThreads, t = i / kLanes, c = 4 * (i % kLanes);
      if (t < kBlock) {
        *reinterpret_cast<float4*>(&s_z[t][c]) = rz[k];
        *reinterpret_cast<float4*>(&s_u[t][c]) = ru[k];
      }
    }
    if (tid < kBlock) {  // in two parts (whose sum is the nearest number): rounded once, a head of one decay would gain the same 2^-25 with every token
      const float2 dec = exp2_fixed_two(to_fixed(rg));
      s_a[tid] = rg == rg ? dec.x : rg;
      s_al[tid] = dec.y;
    }
    __syncthreads();
    if (const int next = t0 + (kEnds ? count : kBlock); next < sq.len) fetch(next);
    {  // x.y, four lanes a token
      for (int t0x = 8 * warp; t0x < kBlock; t0x += 8 * kWarps) {
        const int t = t0x + (lane >> 2);
        float d = 0.f;
        if (t < count)
#pragma unroll 4
          for (int c = 4 * (lane & 3); c < D; c += 16) {
            const float4 p4 = *reinterpret_cast<const float4*>(&s_x[t][c]), q4 = *reinterpret_cast<const float4*>(&s_y[t][c]);
            d = fmaf(p4.x, q4.x, fmaf(p4.y, q4.y, fmaf(p4.z, q4.z, fmaf(p4.w, q4.w, d))));
          }
        d += __shfl_xor_sync(0xffffffffu, d, 1);
        d += __shfl_xor_sync(0xffffffffu, d, 2);
        if (t < count && (lane & 3) == 0) s_d[t] = d;
      }
    }
    auto one = [&](int t) {
      const float dec = s_a[t];
      float2 acc[2] = {f2(0.f, 0.f), f2(0.f, 0.f)};
      if (active) {  // forwards R = a R + y z, read before the write; backwards R = a (R + y z)
        const float4 zv = *reinterpret_cast<const float4*>(&s_z[t][4 * cq]);
        const float wr = rev ? write * (dec + s_al[t]) : write;
        const float2 z0 = f2(wr * zv.x, wr * zv.y), z1 = f2(wr * zv.z, wr * zv.w), dh = f2(dec, dec), dl = f2(s_al[t], s_al[t]);
#pragma unroll
        for (int i0 = 0; i0 < kRows; i0 += 4) {
          const float4 x4 = *reinterpret_cast<const float4*>(&s_x[t][row0 + i0]), y4 = *reinterpret_cast<const float4*>(&s_y[t][row0 + i0]);
          const float xr[4] = {x4.x, x4.y, x4.z, x4.w}, yr[4] = {y4.x, y4.y, y4.z, y4.w};
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const int i = i0 + k;
            const float xv = xr[k], yv = yr[k];
            float2 lo = f2(S[i].x, S[i].y), hi = f2(S[i].z, S[i].w);
            acc[0] = fma2(lo, f2(xv, xv), acc[0]);
            acc[1] = fma2(hi, f2(xv, xv), acc[1]);
            lo = fma2(lo, dh, fma2(lo, dl, mul2(f2(yv, yv), z0)));
            hi = fma2(hi, dh, fma2(hi, dl, mul2(f2(yv, yv), z1)));
            S[i] = make_float4(lo.x, lo.y, hi.x, hi.y);
          }
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
    };
    // Four tokens at a time where there are (and registers for them): only the state passes from one to the next, and their sums' shuffles overlap.
    constexpr int kTogether = kRows > 4 ? 1 : 4;
    if (count == kBlock) {
#pragma unroll kTogether
      for (int t = 0; t < kBlock; ++t) one(t);
    } else {
#pragma unroll 1
      for (int t = 0; t < count; ++t) one(t);
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
        pre *= rev ? read : read * (s_a[t] + s_al[t]);
        const size_t at = (token(t) * H + h) * D + col0 + c;
        const float o = fmaf(pair_scale * s_d[t], s_z[t][c], pre);
        if (out32) static_cast<float*>(out)[at] = o;
        else static_cast<T*>(out)[at] = from_f<T>(o);
        if (u) dot = pre * s_u[t][c];
      }
      if (dots) {
        constexpr int kWidth = kCols < 32 ? kCols : 32;
#pragma unroll
        for (int o = kWidth / 2; o; o >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, o);
        if (c % kWidth == 0) s_dot[t][c / 32] = dot;
      }
    }
    __syncthreads();
    if (dots && tid < count) {
      float dot = 0.f;
#pragma unroll
      for (int i = 0; i < (kCols + 31) / 32; ++i) dot += s_dot[tid][i];
      dots[((size_t)slice * H + h) * geo.total_tokens + token(tid)] = dot;
    }
    if (ends && active && (t0 + count == sq.len || (t0 + count) % span == 0)) {
      float* const to = ends + (entry0 + (size_t)((t0 + count - 1) / span) * H) * D * D + own;
#pragma unroll
      for (int i = 0; i < kRows; ++i) *reinterpret_cast<float4*>(to + (size_t)i * D) = S[i];
    }
  }
  if (active) {
    if (float* const fin = p.fin) {
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

// One or two tokens of a dense batch whose heads fill the SMs: a CTA holds a whole state, and what it writes leaves before its outputs are summed, so
// that a CTA's memory is idle as short as may be.  256 rows of 32 heads of 128, one token: 159 us, the copy rate; 192 with
// the kernel above.
template <int D, typename T>
__global__ void __launch_bounds__(256, D == 128 ? 2 : 4) la_step_kernel(const Call c, const __grid_constant__ Pass p) {
  after_previous();
  constexpr int kLanes = D / 4, kGroups = 256 / kLanes, kRows = D / kGroups;
  const int H = c.geo.heads, n = blockIdx.x / H, h = blockIdx.x - n * H, tid = threadIdx.x, kg = tid / kLanes, cq = tid - kg * kLanes, row0 = kg * kRows;
  const size_t at = (size_t)blockIdx.x * D * D + (size_t)row0 * D + 4 * cq;
  __shared__ __align__(16) float s_x[D], s_y[D], s_part[kGroups][D];
  __shared__ float s_d[D / 32];
  float4 S[kRows];
  if (p.init) {
#pragma unroll
    for (int i = 0; i < kRows; ++i) S[i] = *reinterpret_cast<const float4*>(p.init + at + (size_t)i * D);
  } else {
#pragma unroll
    for (int i = 0; i < kRows; ++i) S[i] = make_float4(0.f, 0.f, 0.f, 0.f);
  }
  for (int t = 0; t < c.geo.seq_len; ++t) {
    const size_t tok = (size_t)n * c.geo.seq_len + t;
    const T* z = static_cast<const T*>(p.z) + (tok * H + h) * D;
    float xv = 0.f, yv = 0.f, zt = 0.f;
    if (tid < D) {
      xv = to_f(static_cast<const T*>(p.x)[(tok * (H / p.x_group) + h / p.x_group) * D + tid]);
      yv = to_f(static_cast<const T*>(p.y)[(tok * (H / p.y_group) + h / p.y_group) * D + tid]);
      zt = to_f(z[tid]);
    }
    const float4 zv = read4(z + 4 * cq);
    const float g = gate(c, tok, h);
    float2 dec = exp2_fixed_two(to_fixed(g));
    if (g != g) dec.x = g;
    if (t > 0) __syncthreads();
    if (tid < D) {
      s_x[tid] = xv;
      s_y[tid] = yv;
      float d = xv * yv;
#pragma unroll
      for (int o = 16; o; o >>= 1) d += __shfl_xor_sync(0xffffffffu, d, o);
      if ((tid & 31) == 0) s_d[tid >> 5] = d;
    }
    __syncthreads();
    float2 acc[2] = {f2(0.f, 0.f), f2(0.f, 0.f)};
    const float2 z0 = f2(p.write * zv.x, p.write * zv.y), z1 = f2(p.write * zv.z, p.write * zv.w), dh = f2(dec.x, dec.x), dl = f2(dec.y, dec.y);
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
      const float xr = s_x[row0 + i], yr = s_y[row0 + i];
      float2 lo = f2(S[i].x, S[i].y), hi = f2(S[i].z, S[i].w);
      acc[0] = fma2(lo, f2(xr, xr), acc[0]);
      acc[1] = fma2(hi, f2(xr, xr), acc[1]);
      lo = fma2(lo, dh, fma2(lo, dl, mul2(f2(yr, yr), z0)));
      hi = fma2(hi, dh, fma2(hi, dl, mul2(f2(yr, yr), z1)));
      S[i] = make_float4(lo.x, lo.y, hi.x, hi.y);
    }
    if (t == c.geo.seq_len - 1 && p.fin) {
#pragma unroll
      for (int i = 0; i < kRows; ++i) *reinterpret_cast<float4*>(p.fin + at + (size_t)i * D) = S[i];
    }
    *reinterpret_cast<float4*>(&s_part[kg][4 * cq]) = make_float4(acc[0].x, acc[0].y, acc[1].x, acc[1].y);
    __syncthreads();
    if (tid < D) {
      float pre = 0.f, d = 0.f;
#pragma unroll
      for (int i = 0; i < kGroups; ++i) pre += s_part[i][tid];
#pragma unroll
      for (int i = 0; i < D / 32; ++i) d += s_d[i];
      static_cast<T*>(p.out)[(tok * H + h) * D + tid] = from_f<T>(fmaf(p.c * d, zt, p.read * (dec.x + dec.y) * pre));
    }
  }
}
// Whether a call goes there: not where heads are split over SMs, whose latency counts then (8 heads of 128: 5.7 us).
bool takes_step(const Call& c, int D) {
  const long long units = (long long)c.geo.n_seqs * c.geo.heads;
  return !c.geo.cu_seqlens && c.geo.seq_len <= 2 && D >= 64 && chain_slices(units, D) == 1;
}
template <int D, typename T> static int launch_step(const Call& c, const Pass& p, cudaStream_t st) {
  begin_stage(kStageLaChain, st);
  const int rc = launch_kernel(la_step_kernel<D, T>, dim3((unsigned)((long long)c.geo.n_seqs * c.geo.heads)), 256, 0, st, c, p);
  end_stage(st);
  return rc;
}
int launch_step(const Call& c, int D, int dtype, const Pass& p, cudaStream_t st) {
  if (dtype == PKDA_BF16) return D == 128 ? launch_step<128, bf16>(c, p, st) : launch_step<64, bf16>(c, p, st);
  return D == 128 ? launch_step<128, float>(c, p, st) : launch_step<64, float>(c, p, st);
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
  const auto kernel = a.e.ends || a.e.X ? la_chain_kernel<D, kCols, T, true> : la_chain_kernel<D, kCols, T, false>;
  const int rc = launch_kernel(kernel, dim3((unsigned)((long long)a.c.geo.n_seqs * a.c.geo.heads * (D / kCols)), n),
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
int chain_x_parts(long long units, int D) {  // (as ChainCfg has it)
  const int cols = chain_cols(units, D), lanes = cols / 4, groups = 256 / lanes < D / 4 ? 256 / lanes : D / 4, warps = lanes * groups / 32;
  return D / cols * (warps ? warps : 1);
}
int launch_chain(const Call& c, int D, int dtype, const Pass* passes, int n, const ChainEnds& ends, cudaStream_t st) {
  ChainParams a;
  a.c = c;
  a.e = ends;
  for (int i = 0; i < n; ++i) a.pass[i] = passes[i];
  const int cols = chain_cols((long long)c.geo.n_seqs * c.geo.heads, D);
  return dtype == PKDA_BF16 ? launch_width<bf16>(a, D, n, cols, st) : launch_width<float>(a, D, n, cols, st);
}

// ------------------------------------------------------------------------------------------------ the gate's gradient
// One CTA per (sequence, segment, head); sums in 64 bits, since the tokens' shares differ in sign.
__device__ __forceinline__ double warp_suffix(double x, int lane) {  // sum over this lane and those behind it
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const double y = __shfl_down_sync(0xffffffffu, x, o);
    if (lane + o < 32) x += y;
  }
  return x;
}

// Of the CTA, the same in every thread.
__device__ __forceinline__ double block_sum(double x, double* s_sum) {
#pragma unroll
  for (int o = 16; o; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) s_sum[threadIdx.x >> 5] = x;
  __syncthreads();
  x = 0.0;
  for (int w = 0; w < 8; ++w) x += s_sum[w];
  return x;
}
__device__ __forceinline__ double inner(const float* S, const float* dS, size_t unit, int D, double* s_sum) {
  double x = 0.0;
  for (int i = threadIdx.x; i < D * D; i += 256) x += (double)S[unit * D * D + i] * (double)dS[unit * D * D + i];
  return block_sum(x, s_sum);
}

// <S, dS> at the end of a segment, in every thread.
__device__ __forceinline__ double end_product(const GateGrad& a, long long entry_head) {
  double x = 0.0;
  for (int i = 0; i < a.x_parts; ++i) x += a.X[entry_head * a.x_parts + i];
  return x;
}

// Behind the token-by-token kernels: a CTA takes a segment of 256 tokens, a thread one of them.  Rows and columns are each off by some 2^-24,
// and their sums from the end on gather that token by token (one sum over 8,192 tokens of strong decay: 1.1e-5 of the result's
// root mean square).  So the sums start anew from <S, dS> at every segment's end, and what they miss it by in front of the segment is taken out in equal steps.
__global__ void __launch_bounds__(256) la_gate_grad_kernel(const GateGrad a) {
  after_previous();
  const Geo& geo = a.c.geo;
  const int H = geo.heads, e = blockIdx.x / H, h = blockIdx.x - e * H;
  int n, seg;
  if (!find_segment(geo, a.segments, e, n, seg)) {
    if (a.part && threadIdx.x == 0) a.part[blockIdx.x] = 0.0;
    return;
  }
  const SeqInfo sq = gdr::sequence(geo, n);
  const int begin = seg * a.segments.chunks * kChunk, end = min(sq.len, begin + a.segments.chunks * kChunk);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, t = begin + tid;
  __shared__ double s_sum[8];
  double mine = 0.0;
  if (begin < end) {
    const bool known = seg > 0 || !a.S0 || a.dS0;
    const double start = seg > 0 ? end_product(a, (long long)blockIdx.x - H)
                                 : a.S0 && a.dS0 ? inner(a.S0, a.dS0, (size_t)n * H + h, a.D, s_sum) : 0.0;
    double x = 0.0;
    if (t < end) {
      const size_t at = (size_t)h * geo.total_tokens + sq.bos + t;
      for (int s = 0; s < a.row_slices; ++s) x += a.row[(size_t)s * H * geo.total_tokens + at];
      for (int s = 0; s < a.col_slices; ++s) x -= a.col[(size_t)s * H * geo.total_tokens + at];
    }
    x = warp_suffix(x, lane);
    __syncthreads();
    if (lane == 0) s_sum[warp] = x;
    __syncthreads();
    double all = end_product(a, blockIdx.x);
    x += all;
    for (int w = 0; w < 8; ++w) {
      if (w > warp) x += s_sum[w];
      all += s_sum[w];
    }
    if (known) x += (start - all) * (end - t) / (end - begin);
    if (t < end) {
      if (a.dg) a.dg[(size_t)(sq.bos + t) * H + h] = (float)x;
      mine = x;
    }
  }
  if (a.part) {
    mine = block_sum(mine, s_sum);
    if (tid == 0) a.part[blockIdx.x] = mine;
  }
}

// Behind the chunked kernels: a CTA takes a segment of up to 1,024 tokens, a thread four of them, a chunk is half a warp.  Rows and
// columns come in coalesced (2 x 2,047 tokens of 12 heads: 25 us with each thread reading its own four).
//
// Rows and columns of a chunk's reads are off by some 2^-19, since their operands are, and the sums from the segment's end on
// gather that chunk by chunk (2.6e-6 of the result's root mean square after one, 1.1e-5 after sixteen, where a token's decay is
// strong).  Two things hold it back.  Where a chunk decays by 2^-kForgets, no pair reaches over it: what reaches over its start is the
// sum of its rows alone, so the sum starts anew, and inside it the columns are added up from its start instead of taken from the
// whole (which is what it says for their sum to be the end); not in a sequence with a decay above 1 anywhere, which may make up for it.  And <S, dS> at the segment's start is known too (it is the end of the segment in front): what the
// sums miss it by is taken out in equal steps over the chunks from the last new start to there.
constexpr double kForgets = 24.0;
__global__ void __launch_bounds__(256) la_gate_chunks_kernel(const GateGrad a) {
  after_previous();
  const Geo& geo = a.c.geo;
  const int H = geo.heads, e = blockIdx.x / H, h = blockIdx.x - e * H;
  int n, seg;
  if (!find_segment(geo, a.segments, e, n, seg)) {
    if (a.part && threadIdx.x == 0) a.part[blockIdx.x] = 0.0;
    return;
  }
  const SeqInfo sq = gdr::sequence(geo, n);
  const int begin = seg * a.segments.chunks * kChunk, end = min(sq.len, begin + a.segments.chunks * kChunk);
  const int tid = threadIdx.x, chunks = max((end - begin + kChunk - 1) / kChunk, 0), mychunk = tid >> 4;
  __shared__ double s_sum[8], s_row[16], s_over[16], s_end[16], s_step[16];
  __shared__ float s_decay[16];
  __shared__ double s_net[1024];  // rows less columns
  __shared__ float s_rows[1024], s_gate[1024];
  const size_t slice = (size_t)H * geo.total_tokens;
  for (int i = tid; begin + i < end; i += 256) {
    const size_t at = (size_t)h * geo.total_tokens + sq.bos + begin + i;
    double row = 0.0, col = 0.0;
#pragma unroll 4
    for (int s = 0; s < a.row_slices; ++s) row += a.row[s * slice + at];
#pragma unroll 5
    for (int s = 0; s < a.col_slices; ++s) col += a.col[s * slice + at];
    s_rows[i] = (float)row;
    s_net[i] = (double)(float)row - col;
    s_gate[i] = gate(a.c, (size_t)(sq.bos + begin + i), h);
  }
  __syncthreads();
  double net[4], rows = 0.0, all = 0.0;
  float decay = 0.f;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int i = 4 * tid + j;
    net[j] = 0.0;
    if (begin + i < end) {
      net[j] = s_net[i];
      rows += s_rows[i];
      decay += s_gate[i];
    }
    all += net[j];
  }
  // suffix sums of the thread's tokens and behind it in its chunk
  double behind = all;
#pragma unroll
  for (int o = 1; o < 16; o <<= 1) {
    const double y = __shfl_down_sync(0xffffffffu, behind, o, 16);
    if ((tid & 15) + o < 16) behind += y;
  }
#pragma unroll
  for (int o = 8; o; o >>= 1) {
    rows += __shfl_xor_sync(0xffffffffu, rows, o, 16);
    decay += __shfl_xor_sync(0xffffffffu, decay, o, 16);
  }
  if ((tid & 15) == 0) {
    s_row[mychunk] = rows;
    s_over[mychunk] = behind;
    s_decay[mychunk] = decay;
  }
  double start = 0.0;  // <S, dS> in front of the segment
  const bool known = seg > 0 || !a.S0 || a.dS0;
  int grows = 0;
  const int* const flags = a.grows + (size_t)first_entry(geo, a.segments, n) * H + h;  // of the sequence's segments, H apart
  for (int s = tid; s < (sq.nchunks + a.segments.chunks - 1) / a.segments.chunks; s += 256) grows |= flags[(size_t)s * H];
  grows = __syncthreads_or(grows);
  if (seg == 0 && a.S0 && a.dS0 && chunks) start = inner(a.S0, a.dS0, (size_t)n * H + h, a.D, s_sum);
  if (tid == 0 && chunks) {
    const float* X = a.X + (size_t)blockIdx.x * a.x_parts;
    double x = 0.0;
    for (int i = 0; i < a.x_parts; ++i) x += X[i];
    if (seg > 0)
      for (int i = 0; i < a.x_parts; ++i) start += X[(long long)i - (long long)H * a.x_parts];
    int anew = chunks;  // the chunks in front of this one are summed from one start
    for (int c = chunks - 1; c >= 0; --c) {
      s_end[c] = x;
      s_step[c] = 0.0;
      if (!grows && (double)s_decay[c] * -1.4426950408889634 > kForgets) {
        s_end[c] = s_row[c] - s_over[c];  // (which makes the sum at the chunk's start that of its rows)
        x = s_row[c];
        anew = c;
      } else {
        x += s_over[c];
      }
    }
    if (known && anew > 0) {
      const double step = (start - x) / anew;
      for (int c = anew - 1; c >= 0; --c) {
        s_end[c] += step * (anew - 1 - c);
        s_step[c] = step;
      }
    }
  }
  __syncthreads();
  double mine = 0.0;
  if (mychunk < chunks) {
    double x = s_end[mychunk] + behind - all;
#pragma unroll
    for (int j = 3; j >= 0; --j) {
      const int t = begin + 4 * tid + j;
      x += net[j];
      if (t < end) {
        const double dg = x + s_step[mychunk] * (kChunk - (4 * (tid & 15) + j)) * (1.0 / kChunk);
        if (a.dg) a.dg[(size_t)(sq.bos + t) * H + h] = (float)dg;
        mine += dg;
      }
    }
  }
  if (a.part) {
    mine = block_sum(mine, s_sum);
    if (tid == 0) a.part[blockIdx.x] = mine;
  }
}

// One CTA a head: the segments' sums in a fixed order.
__global__ void __launch_bounds__(256) la_gate_sum_kernel(const double* part, long long entries, int heads, float* dg) {
  after_previous();
  const int h = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  __shared__ double s_sum[8];
  double x = 0.0;
  for (long long i = threadIdx.x; i < entries; i += 256) x += part[i * heads + h];
#pragma unroll
  for (int o = 16; o; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
  if (lane == 0) s_sum[warp] = x;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < 8; ++w) x += s_sum[w];
    dg[h] = (float)x;
  }
}

int launch_gate_grad(const GateGrad& a, cudaStream_t st) {
  const int H = a.c.geo.heads;
  begin_stage(kStageLaGate, st);
  int rc = launch_kernel(a.grows ? la_gate_chunks_kernel : la_gate_grad_kernel, dim3((unsigned)(a.segments.entries * H)), 256, 0, st, a);
  end_stage(st);
  if (rc != PKDA_OK || !a.part) return rc;
  begin_stage(kStageLaGate, st);
  rc = launch_kernel(la_gate_sum_kernel, H, 256, 0, st, a.part, a.segments.entries, H, a.dg_head);
  end_stage(st);
  return rc;
}

// ------------------------------------------------------------------------------------------------ shared key heads
// blockIdx.y: dq or dk.  Bound by its bytes, the value heads' gradients in fp32.
struct GroupSum {
  const float4* part[2];
  void* out[2];
};
template <typename T>
__global__ void __launch_bounds__(256) la_group_sum_kernel(const GroupSum a, long long quads, int group, int log_row) {
  after_previous();
  const float4* part = a.part[blockIdx.y];
  void* const out = a.out[blockIdx.y];
  const int per_row = 1 << log_row;
  for (long long i = blockIdx.x * 256ll + threadIdx.x; i < quads; i += gridDim.x * 256ll) {
    const long long row = i >> log_row;  // (token, key head)
    const float4* at = part + ((row * group) << log_row) + (i & (per_row - 1));
    float4 s = __ldcs(at);
    for (int j = 1; j < group; ++j) {
      const float4 x = __ldcs(at + ((size_t)j << log_row));
      s.x += x.x; s.y += x.y; s.z += x.z; s.w += x.w;
    }
    if constexpr (sizeof(T) == 4) static_cast<float4*>(out)[i] = s;
    else static_cast<uint2*>(out)[i] = make_uint2(pack_bf16(s.x, s.y), pack_bf16(s.z, s.w));
  }
}
int launch_group_sum(const float* part0, void* out0, const float* part1, void* out1, int dtype, long long tokens, int key_heads, int group, int D,
                     cudaStream_t st) {
  const long long quads = tokens * key_heads * (D / 4);
  int log_row = 0;
  while (4 << log_row < D) ++log_row;
  const dim3 grid((unsigned)(quads < 256ll * 8 * sm_count() ? (quads + 255) / 256 : 8ll * sm_count()), 2);
  const GroupSum a = {{reinterpret_cast<const float4*>(part0), reinterpret_cast<const float4*>(part1)}, {out0, out1}};
  begin_stage(kStageLaGroup, st);
  const int rc = dtype == PKDA_BF16 ? launch_kernel(la_group_sum_kernel<bf16>, grid, 256, 0, st, a, quads, group, log_row)
                                    : launch_kernel(la_group_sum_kernel<float>, grid, 256, 0, st, a, quads, group, log_row);
  end_stage(st);
  return rc;
}

}  // namespace la
}  // namespace pkda
