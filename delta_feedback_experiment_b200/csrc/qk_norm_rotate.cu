// RMS norm of every head's queries and keys with a learned weight, and the rotation by the token's position, in one pass:
//   r = 1 / sqrt(mean(x^2) + eps),   n = x r w,   (a, b) -> (a cos - b sin, b cos + a sin) for each pair of channels
// and backwards, with h = dy rotated back,
//   dw = sum h x r,   dx = r (h w) - x r^3 mean(h w x).
// Nothing is kept for the backward: what it needs of x it reads anyway.  Bytes: x in and y out, or x and dy in and dx out.  8 x 4,096 tokens of
// 32 heads of 128, bf16: forward 102 us (5.3 TB/s), backward 161 (5.0).  Instruction slots stand in front of the memory: packed arithmetic,
// cosines and sines where no bank is met twice, and positions asked for an item ahead took it there from 120 and 179; 24 instead of 16 warps
// an SM in the forward leave 84 registers a thread and 113 us.
//
// A few adjacent lanes share a row; a lane holds two vectors of it whose elements are each other's partners, so that the rotation
// stays in the lane.  The rows of a warp are heads of one token (of several where there are few heads): the token's cosines and sines are formed once,
// a few by each lane, and passed through shared memory.
//
// Angles.  position * inv_freq is a whole number of turns and a rest, and only the rest counts: inv_freq / 2 pi as a 64-bit binary
// fraction times the position, modulo 2^64, is that rest for a position of any size, where a product in 32 bits is off by a tenth at a
// position of a million.  Its upper 32 bits, less the nearest quarter turn, go to fp32.  The fraction is off by a unit of its last place, so
// an angle by |position| * 2^-64 turns: less than fp32 tells apart up to positions of 2^39.
#include "pkda_common.cuh"
#include "pkda_launch.h"

#include <type_traits>

namespace pkda {
namespace rotate {

constexpr int kThreads = 256, kWarps = kThreads / 32, kMaxHalf = 128;
constexpr int kTable = 256;  // cosines and sines of a warp's tokens: tokens * head_dim / 2, at most 32 lanes * 8 elements

template <typename T, int N> struct Vec;
template <> struct Vec<bf16, 8> { uint4 r; };
template <> struct Vec<float, 4> { float4 r; };
template <typename T> struct Vec<T, 1> { T r; };
__device__ __forceinline__ void widen(const Vec<bf16, 8>& v, float (&f)[8]) {
  const uint32_t w[4] = {v.r.x, v.r.y, v.r.z, v.r.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 p = unpack_bf16(w[i]);
    f[2 * i] = p.x;
    f[2 * i + 1] = p.y;
  }
}
__device__ __forceinline__ void widen(const Vec<float, 4>& v, float (&f)[4]) { f[0] = v.r.x; f[1] = v.r.y; f[2] = v.r.z; f[3] = v.r.w; }
template <typename T> __device__ __forceinline__ void widen(const Vec<T, 1>& v, float (&f)[1]) { f[0] = to_f(v.r); }
__device__ __forceinline__ void narrow(const float (&f)[8], Vec<bf16, 8>& v) {
  v.r = make_uint4(pack_bf16(f[0], f[1]), pack_bf16(f[2], f[3]), pack_bf16(f[4], f[5]), pack_bf16(f[6], f[7]));
}
__device__ __forceinline__ void narrow(const float (&f)[4], Vec<float, 4>& v) { v.r = make_float4(f[0], f[1], f[2], f[3]); }
template <typename T> __device__ __forceinline__ void narrow(const float (&f)[1], Vec<T, 1>& v) { v.r = from_f<T>(f[0]); }

struct Params {
  pkda_qk_rotate_args a;
  int tokens_warp[2];  // tokens that a warp takes at once, a power of two
  int parts[2];        // into how many items the heads of a token are split
  float* part;         // [2][gridDim.x][head_dim], the weights' gradients of each CTA
};

// What a lane holds of one row: the partners e0.. and e1.. of `it`.
template <int VEC, int LPR, bool kInter> struct Lane {
  int e0, e1, pair;  // first elements, and the pairs' index
  bool live;
  __device__ __forceinline__ Lane(int lane, int it, int D, int half) {
    const int p = (lane % LPR + LPR * it) * VEC;
    live = p < D / 2;
    pair = p;
    if (kInter) {
      e0 = 2 * p;
      e1 = e0 + VEC;
    } else if (p < half) {
      e0 = p;
      e1 = p + half;
    } else {
      e0 = half + p;
      e1 = e0 + D / 2 - half;
    }
  }
};
// Neighbouring elements to partners and back.
template <int VEC, bool kInter> __device__ __forceinline__ void part_pairs(float (&a)[VEC], float (&b)[VEC]) {
  if constexpr (kInter && VEC > 1) {
    float e[2 * VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      e[j] = a[j];
      e[VEC + j] = b[j];
    }
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      a[j] = e[2 * j];
      b[j] = e[2 * j + 1];
    }
  }
}
template <int VEC, bool kInter> __device__ __forceinline__ void join_pairs(float (&a)[VEC], float (&b)[VEC]) {
  if constexpr (kInter && VEC > 1) {
    float e[2 * VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      e[2 * j] = a[j];
      e[2 * j + 1] = b[j];
    }
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      a[j] = e[j];
      b[j] = e[VEC + j];
    }
  }
}

// Rows on their way, in shared memory: a lane's own two vectors (and two of dy) of each turn of its warp, whatever token the turn is of.
// (The path of single elements keeps one row ahead in registers.)
constexpr int kSlots = 4, kAhead = kSlots - 1;
template <int VEC, bool kBwd> constexpr int rows_bytes() { return VEC == 1 ? 0 : kWarps * kSlots * (kBwd ? 4 : 2) * 32 * 16; }
__device__ __forceinline__ void rows_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(kAhead - 1) : "memory"); }
__device__ __forceinline__ void rows_asked() { asm volatile("cp.async.commit_group;" ::: "memory"); }

// blockIdx.y: the queries or the keys, so that a lane's part of the weight and of its gradient stay in registers.
template <typename T, int VEC, int LPR, int ITER, bool kInter, bool kBwd>
__global__ void __launch_bounds__(kThreads, 2) qk_rotate_kernel(const __grid_constant__ Params q) {
  after_previous();
  const pkda_qk_rotate_args& a = q.a;
  const int w = blockIdx.y, H = a.heads[w];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, D = a.head_dim, half = a.inv_freq ? a.half : 0, pairs = D / 2;
  __shared__ unsigned long long s_turn[kMaxHalf];
  __shared__ __align__(16) float s_cos[kWarps][kTable], s_sin[kWarps][kTable];
  __shared__ float s_dw[kBwd ? kWarps : 1][kBwd ? 256 : 1];
  for (int j = tid; j < half; j += kThreads) {  // turns of one position, less whole ones, in units of 2^-64: 1 / 2 pi in two parts
    constexpr double kTurn = 0x1.45f306dc9c883p-3, kTurnLo = -0x1.6b01ec5417056p-57;
    const double f = (double)a.inv_freq[j], hi = f * kTurn, lo = fma(f, kTurn, -hi) + f * kTurnLo;
    s_turn[j] = __double2ull_rn((hi - floor(hi)) * 0x1p64) + (unsigned long long)__double2ll_rn((lo - rint(lo)) * 0x1p64);
  }
  float *const cosines = s_cos[warp], *const sines = s_sin[warp];
  for (int i = lane; i < kTable; i += 32) {  // (what does not turn keeps this)
    cosines[i] = 1.f;
    sines[i] = 0.f;
  }
  // Where pair j of a token lies: a lane's eight in two fours, those of its neighbours beside them, so that a read meets every bank once.
  auto place = [&](int j) { return VEC == 8 ? (j & 4 ? pairs >> 1 : 0) + (j >> 3) * 4 + (j & 3) : j; };
  __syncthreads();
  const int tw = q.tokens_warp[w], log_tw = 31 - __clz(tw), heads_warp = 32 / LPR / tw, group = lane / LPR;
  const int ts = group / heads_warp, hs = group - ts * heads_warp;  // this lane's token and head of the warp's
  constexpr bool kAsync = VEC > 1;
  const int parts = q.parts[w], turns = (H + heads_warp - 1) / heads_warp, per = (turns + parts - 1) / parts;
  const long long tokens = (long long)a.batch * a.tokens, items = H ? (tokens + tw - 1) / tw * parts : 0;
  const long long step = (long long)gridDim.x * kWarps;
  float wa[ITER][VEC], wb[ITER][VEC], dwa[ITER][VEC], dwb[ITER][VEC];
#pragma unroll
  for (int it = 0; it < ITER; ++it) {
    const Lane<VEC, LPR, kInter> l(lane, it, D, half);
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      wa[it][j] = a.weight[w] && l.live ? a.weight[w][l.e0 + j] : 1.f;
      wb[it][j] = a.weight[w] && l.live ? a.weight[w][l.e1 + j] : 1.f;
      dwa[it][j] = dwb[it][j] = 0.f;
    }
    part_pairs<VEC, kInter>(wa[it], wb[it]);
  }
  const float inv_d = 1.f / (float)D;

  // A place in the warp's work: an item is some heads of tw tokens (no item is without any).
  struct Place {
    long long item, tok;
    int turn, last;
    const T *x, *dy;
  };
  auto enter = [&](Place& at, long long item) {
    const long long block = parts == 1 ? item : item / parts;
    at.item = item;
    at.turn = (int)(item - block * parts) * per;
    at.last = min(at.turn + per, turns);
    at.tok = block * tw + ts;
    const unsigned b = (unsigned)at.tok / (unsigned)a.tokens, t = (unsigned)at.tok - b * (unsigned)a.tokens;  // (fewer than 2^31 tokens)
    at.x = static_cast<const T*>(a.x[w]) + b * a.x_stride[w][0] + t * a.x_stride[w][1];
    at.dy = kBwd ? static_cast<const T*>(a.dy[w]) + b * a.dy_stride[w][0] + t * a.dy_stride[w][1] : nullptr;
  };
  extern __shared__ __align__(16) uint4 s_rows[];
  constexpr int kVecs = kBwd ? 4 : 2;
  uint4* const mine = s_rows + warp * kSlots * kVecs * 32 + lane;
  Place ask = {};
  const Lane<VEC, LPR, kInter> lane0(lane, 0, D, half);
  auto ask_row = [&](int slot) {  // the next row of the warp's that nobody has asked for
    if (ask.item < items) {
      const int h = ask.turn * heads_warp + hs;
      const bool on = ask.tok < tokens && h < H && lane0.live;
      const T* p = on ? ask.x + h * a.x_stride[w][2] : static_cast<const T*>(a.x[w]);
      uint4* to = mine + slot * kVecs * 32;
      cp_async16(to, on ? p + lane0.e0 : p, on);
      cp_async16(to + 32, on ? p + lane0.e1 : p, on);
      if (kBwd) {
        const T* d = on ? ask.dy + h * a.dy_stride[w][2] : static_cast<const T*>(a.dy[w]);
        cp_async16(to + 64, on ? d + lane0.e0 : d, on);
        cp_async16(to + 96, on ? d + lane0.e1 : d, on);
      }
      if (++ask.turn >= ask.last) {
        if (ask.item + step < items) enter(ask, ask.item + step);
        else ask.item = items;
      }
    }
    rows_asked();
  };
  // The position that this lane turns pairs of (tw is a power of two: every 32nd pair is of the same token), asked for an item ahead.
  auto position_of = [&](long long item) -> unsigned long long {
    const long long tk = (parts == 1 ? item : item / parts) * tw + (lane & (tw - 1));
    if (tk >= tokens) return 0;
    const unsigned b = (unsigned)tk / (unsigned)a.tokens, t = (unsigned)tk - b * (unsigned)a.tokens;
    const long long where = b * (long long)a.position_row + t;
    return !a.positions ? t : a.positions64 ? static_cast<const long long*>(a.positions)[where] : (long long)static_cast<const int*>(a.positions)[where];
  };
  unsigned long long position = 0;
  int slot = 0;
  const long long first_item = (long long)blockIdx.x * kWarps + warp;
  ask.item = first_item;
  if (kAsync && ask.item < items) {
    enter(ask, ask.item);
#pragma unroll
    for (int i = 0; i < kAhead; ++i) ask_row(i);
  }

  if (half && first_item < items) position = position_of(first_item);
  for (long long item = first_item; item < items; item += step) {
    Place now;
    enter(now, item);
    const long long tok = now.tok;
    const int first = now.turn, last = now.last;
    const T *x = now.x, *dy = now.dy;
    // Rows that are not there are zeros, and add zeros to the weights' gradients as long as their r is a number: without eps too.
    const int heads = tok < tokens ? H : 0;
    T* y = static_cast<T*>(kBwd ? a.dx[w] : a.y[w]) + tok * H * D;
    Vec<T, VEC> raw[ITER][2], drw[ITER][2];
    auto load = [&](int turn) {
      const int h = turn * heads_warp + hs;
#pragma unroll
      for (int it = 0; it < ITER; ++it) {
        const Lane<VEC, LPR, kInter> l(lane, it, D, half);
        raw[it][0] = raw[it][1] = Vec<T, VEC>{};
        if (kBwd) drw[it][0] = drw[it][1] = Vec<T, VEC>{};
        if (turn < last && tok < tokens && h < H && l.live) {
          const T* p = x + h * a.x_stride[w][2];
          raw[it][0] = *reinterpret_cast<const Vec<T, VEC>*>(p + l.e0);
          raw[it][1] = *reinterpret_cast<const Vec<T, VEC>*>(p + l.e1);
          if (kBwd) {
            const T* d = dy + h * a.dy_stride[w][2];
            drw[it][0] = *reinterpret_cast<const Vec<T, VEC>*>(d + l.e0);
            drw[it][1] = *reinterpret_cast<const Vec<T, VEC>*>(d + l.e1);
          }
        }
      }
    };
    if (!kAsync) load(first);
    if (half) {  // the tokens' cosines and sines, while the first rows come
      __syncwarp();
      const unsigned long long pos = position;
      if (item + step < items) position = position_of(item + step);
#pragma unroll 2
      for (int i = lane; i < half << log_tw; i += 32) {
        const int t = i & (tw - 1), j = i >> log_tw;
        const unsigned rest = (unsigned)((pos * s_turn[j]) >> 32), quarter = (rest + 0x20000000u) >> 30;
        float s, c;
        sincospif((float)(int)(rest - (quarter << 30)) * 4.656612873077393e-10f, &s, &c);  // (2^-31 half turns)
        if (quarter & 1) {
          const float x = s;
          s = c;
          c = -x;
        }
        if (quarter & 2) {
          s = -s;
          c = -c;
        }
        cosines[t * pairs + place(j)] = c;
        sines[t * pairs + place(j)] = s;
      }
      __syncwarp();
    }
    for (int turn = first; turn < last; ++turn) {
      const int h = turn * heads_warp + hs;
      float xa[ITER][VEC], xb[ITER][VEC], ga[ITER][VEC], gb[ITER][VEC];  // backwards g is dy rotated back
      constexpr int N = ITER * VEC;                                      // (taken two at a time: packed arithmetic)
      auto two = [](const float (&m)[ITER][VEC], int k) { return f2(m[k / VEC][k % VEC], m[(k + 1) / VEC][(k + 1) % VEC]); };
      auto put = [](float (&m)[ITER][VEC], int k, float2 v) {
        m[k / VEC][k % VEC] = v.x;
        m[(k + 1) / VEC][(k + 1) % VEC] = v.y;
      };
      float co[ITER][VEC], si[ITER][VEC];
      auto angles = [&]() {
        if constexpr (VEC == 1) {
#pragma unroll
          for (int it = 0; it < ITER; ++it) {
            const Lane<VEC, LPR, kInter> l(lane, it, D, half);
            const int at = ts * pairs + (l.live ? l.pair : 0);
            co[it][0] = cosines[at];
            si[it][0] = sines[at];
          }
        } else {
          const int at = ts * pairs + (lane0.live ? lane0.pair / VEC * 4 : 0);
#pragma unroll
          for (int j = 0; j < VEC; j += 4) {
            const float4 c = *reinterpret_cast<const float4*>(cosines + at + (j ? pairs >> 1 : 0));
            const float4 s = *reinterpret_cast<const float4*>(sines + at + (j ? pairs >> 1 : 0));
            co[0][j] = c.x; co[0][j + 1] = c.y; co[0][j + 2] = c.z; co[0][j + 3] = c.w;
            si[0][j] = s.x; si[0][j + 1] = s.y; si[0][j + 2] = s.z; si[0][j + 3] = s.w;
          }
        }
      };
      if constexpr (kAsync) {
        rows_wait();
        const uint4* from = mine + slot * kVecs * 32;
        const auto take = [](const uint4& v) {
          Vec<T, VEC> r;
          *reinterpret_cast<uint4*>(&r) = v;
          return r;
        };
        raw[0][0] = take(from[0]);
        raw[0][1] = take(from[32]);
        if (kBwd) {
          drw[0][0] = take(from[64]);
          drw[0][1] = take(from[96]);
        }
        ask_row((slot + kAhead) % kSlots);  // where the turn before had its row, which has left for memory
        slot = (slot + 1) % kSlots;
      }
#pragma unroll
      for (int it = 0; it < ITER; ++it) {
        widen(raw[it][0], xa[it]);
        widen(raw[it][1], xb[it]);
        part_pairs<VEC, kInter>(xa[it], xb[it]);
        if constexpr (kBwd) {
          widen(drw[it][0], ga[it]);
          widen(drw[it][1], gb[it]);
          part_pairs<VEC, kInter>(ga[it], gb[it]);
        }
      }
      if (!kAsync) load(turn + 1);  // into the same registers, a row ahead
      const float2 minus = f2(-1.f, -1.f);
      float2 ss2 = f2(0.f, 0.f), m2 = f2(0.f, 0.f);
      if (kBwd) angles();
#pragma unroll
      for (int k = 0; k < N; k += 2) {
        const float2 a2 = two(xa, k), b2 = two(xb, k);
        ss2 = fma2(a2, a2, ss2);
        ss2 = fma2(b2, b2, ss2);
        if constexpr (kBwd) {
          const float2 c = two(co, k), s = two(si, k), da = two(ga, k), db = two(gb, k);
          const float2 g0 = fma2(db, s, mul2(da, c)), g1 = fma2(mul2(da, minus), s, mul2(db, c));
          put(ga, k, g0);
          put(gb, k, g1);
          m2 = fma2(mul2(g0, two(wa, k)), a2, m2);
          m2 = fma2(mul2(g1, two(wb, k)), b2, m2);
        }
      }
      float ss = ss2.x + ss2.y, m = m2.x + m2.y;
#pragma unroll
      for (int o = LPR / 2; o; o >>= 1) {
        ss += __shfl_xor_sync(0xffffffffu, ss, o);
        if (kBwd) m += __shfl_xor_sync(0xffffffffu, m, o);
      }
      const float r = 1.f / sqrtf(ss * inv_d + (!kBwd || h < heads ? a.eps : 1.f));
      const float2 r2 = f2(r, r);
      float oas[ITER][VEC], obs[ITER][VEC];
      if (!kBwd) angles();
      [[maybe_unused]] const float f = -(r * m * inv_d) * (r * r);  // (r m is of the size of dy: r^3 alone leaves fp32's range for rows of 2^43)
#pragma unroll
      for (int k = 0; k < N; k += 2) {
        const float2 a2 = two(xa, k), b2 = two(xb, k);
        if constexpr (kBwd) {
          const float2 ha = mul2(two(ga, k), r2), hb = mul2(two(gb, k), r2);
          put(dwa, k, fma2(ha, a2, two(dwa, k)));
          put(dwb, k, fma2(hb, b2, two(dwb, k)));
          put(oas, k, fma2(ha, two(wa, k), mul2(a2, f2(f, f))));
          put(obs, k, fma2(hb, two(wb, k), mul2(b2, f2(f, f))));
        } else {
          const float2 c = two(co, k), s = two(si, k);
          const float2 na = mul2(mul2(a2, r2), two(wa, k)), nb = mul2(mul2(b2, r2), two(wb, k));
          put(oas, k, fma2(mul2(nb, minus), s, mul2(na, c)));
          put(obs, k, fma2(na, s, mul2(nb, c)));
        }
      }
#pragma unroll
      for (int it = 0; it < ITER; ++it) {
        const Lane<VEC, LPR, kInter> l(lane, it, D, half);
        float (&oa)[VEC] = oas[it], (&ob)[VEC] = obs[it];
        join_pairs<VEC, kInter>(oa, ob);
        if (h < heads && l.live) {
          Vec<T, VEC> v0, v1;
          narrow(oa, v0);
          narrow(ob, v1);
          T* p = y + (long long)h * D;
          *reinterpret_cast<Vec<T, VEC>*>(p + l.e0) = v0;
          *reinterpret_cast<Vec<T, VEC>*>(p + l.e1) = v1;
        }
      }
    }
  }

  if constexpr (kBwd) {
    if (!a.dweight[w]) return;
    // the CTA's sums: rows of a warp by shuffles, then the warps one after another
#pragma unroll
    for (int it = 0; it < ITER; ++it) {
      const Lane<VEC, LPR, kInter> l(lane, it, D, half);
#pragma unroll
      for (int j = 0; j < VEC; ++j)
#pragma unroll
        for (int o = 16; o >= LPR; o >>= 1) {
          dwa[it][j] += __shfl_xor_sync(0xffffffffu, dwa[it][j], o);
          dwb[it][j] += __shfl_xor_sync(0xffffffffu, dwb[it][j], o);
        }
      join_pairs<VEC, kInter>(dwa[it], dwb[it]);
      if (lane < LPR && l.live) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          s_dw[warp][l.e0 + j] = dwa[it][j];
          s_dw[warp][l.e1 + j] = dwb[it][j];
        }
      }
    }
    __syncthreads();
    for (int c = tid; c < D; c += kThreads) {
      float x = 0.f;
      for (int i = 0; i < kWarps; ++i) x += s_dw[i][c];
      q.part[((size_t)w * gridDim.x + blockIdx.x) * D + c] = x;
    }
  }
}

// One CTA per (tensor, 32 channels): the CTAs' sums in a fixed order.
__global__ void __launch_bounds__(256) qk_rotate_dw_kernel(const float* part, int ctas, int D, float* dw0, float* dw1) {
  after_previous();
  const int w = blockIdx.y, c = blockIdx.x * 32 + (threadIdx.x & 31), i0 = threadIdx.x >> 5;
  float* dw = w ? dw1 : dw0;
  __shared__ float s[8][32];
  float x = 0.f;
  if (dw && c < D)
    for (int i = i0; i < ctas; i += 8) x += part[((size_t)w * ctas + i) * D + c];
  s[i0][threadIdx.x & 31] = x;
  __syncthreads();
  if (i0 == 0 && dw && c < D) {
    for (int i = 1; i < 8; ++i) x += s[i][threadIdx.x];
    dw[c] = x;
  }
}

static int check(const pkda_qk_rotate_args& a, bool bwd) {
  if (a.batch < 0 || a.tokens < 0 || a.heads[0] < 0 || a.heads[1] < 0) return PKDA_ERR_SHAPE;
  if (a.head_dim < 2 || a.head_dim > 256 || a.head_dim % 2 || a.half < 0 || 2 * a.half > a.head_dim) return PKDA_ERR_SHAPE;
  if ((long long)a.batch * a.tokens > (1ll << 31) - 1) return PKDA_ERR_SHAPE;
  if (a.dtype != PKDA_BF16 && a.dtype != PKDA_F32) return PKDA_ERR_DTYPE;
  if (a.batch == 0 || a.tokens == 0) return PKDA_OK;
  const uintptr_t size = a.dtype == PKDA_BF16 ? 2 : 4;
  for (int w = 0; w < 2; ++w) {
    if (a.heads[w] == 0) continue;
    if (!a.x[w] || (bwd ? !a.dy[w] || !a.dx[w] : !a.y[w])) return PKDA_ERR_NULL;
    if (!aligned({a.x[w], a.y[w], a.dy[w], a.dx[w]}, size)) return PKDA_ERR_ALIGN;
  }
  if (!aligned({a.weight[0], a.weight[1], a.inv_freq, a.dweight[0], a.dweight[1]}, 4) || !aligned({a.positions}, a.positions64 ? 8 : 4))
    return PKDA_ERR_ALIGN;
  return PKDA_OK;
}

// Whether rows can be moved 16 bytes at a time, partners in lanes.
static bool wide(const pkda_qk_rotate_args& a, bool bwd) {
  const int vec = a.dtype == PKDA_BF16 ? 8 : 4, D = a.head_dim, half = a.inv_freq ? a.half : 0;
  if (D % (2 * vec) || (!a.interleaved && half % vec)) return false;
  for (int w = 0; w < 2; ++w) {
    if (!a.heads[w]) continue;
    if (!aligned({a.x[w], bwd ? a.dy[w] : a.y[w], bwd ? a.dx[w] : nullptr}, 16)) return false;
    for (int i = 0; i < 3; ++i)
      if (a.x_stride[w][i] % vec || (bwd && a.dy_stride[w][i] % vec)) return false;
  }
  return true;
}

constexpr int kCtasPerSm = 2;  // of each tensor's, twice what is resident at most
static int most_ctas() { return kCtasPerSm * sm_count(); }

template <typename T, int VEC, int LPR, int ITER, bool kInter, bool kBwd> static int launch(Params& q, cudaStream_t st) {
  const pkda_qk_rotate_args& a = q.a;
  const int rows = 32 / LPR;
  const long long tokens = (long long)a.batch * a.tokens, warps = (long long)most_ctas() * kWarps;
  long long ctas = 1;
  for (int w = 0; w < 2; ++w) {
    int& tw = q.tokens_warp[w];
    for (tw = 1; tw < rows && rows / tw >= 2 * a.heads[w]; tw *= 2) {}
    const int hw = rows / tw, turns = (a.heads[w] + hw - 1) / hw;
    const long long blocks = (tokens + tw - 1) / tw;
    long long parts = blocks >= warps ? 1 : warps / blocks;
    if (parts > turns) parts = turns;
    if (parts < 1) parts = 1;
    if (turns > 0) parts = (turns + (turns + parts - 1) / parts - 1) / ((turns + parts - 1) / parts);  // (none without heads)
    q.parts[w] = (int)parts;
    const long long n = (blocks * q.parts[w] + kWarps - 1) / kWarps;
    if (n > ctas) ctas = n;
  }
  const int grid = (int)(ctas < most_ctas() ? ctas : most_ctas());
  q.part = static_cast<float*>(a.workspace);
  begin_stage(kBwd ? kStageQkRotateBwd : kStageQkRotateFwd, st);
  const auto kernel = qk_rotate_kernel<T, VEC, LPR, ITER, kInter, kBwd>;
  if (!ensure_dynamic_smem(kernel, rows_bytes<VEC, kBwd>())) return PKDA_ERR_LAUNCH;
  int rc = launch_kernel(kernel, dim3(grid, 2), kThreads, rows_bytes<VEC, kBwd>(), st, q);
  end_stage(st);
  if (!kBwd || rc != PKDA_OK || !(a.dweight[0] || a.dweight[1])) return rc;
  begin_stage(kStageQkRotateDw, st);
  const float* part = q.part;
  rc = launch_kernel(qk_rotate_dw_kernel, dim3((a.head_dim + 31) / 32, 2), 256, 0, st, part, grid, a.head_dim, a.dweight[0], a.dweight[1]);
  end_stage(st);
  return rc;
}

template <typename T, bool kInter, bool kBwd> static int launch_rows(Params& q, cudaStream_t st) {
  constexpr int VEC = 16 / sizeof(T);
  if (!wide(q.a, kBwd)) return launch<T, 1, 32, kMaxHalf / 32, kInter, kBwd>(q, st);
  const int lanes = q.a.head_dim / 2 / VEC;
  if (lanes <= 4) return launch<T, VEC, 4, 1, kInter, kBwd>(q, st);
  if (lanes <= 8) return launch<T, VEC, 8, 1, kInter, kBwd>(q, st);
  if constexpr (sizeof(T) == 4)
    if (lanes > 16) return launch<T, VEC, 32, 1, kInter, kBwd>(q, st);
  return launch<T, VEC, 16, 1, kInter, kBwd>(q, st);
}

template <bool kBwd> static int run(const pkda_qk_rotate_args* a, cudaStream_t st) {
  if (int rc = check(*a, kBwd)) return rc;
  Params q;
  q.a = *a;
  if (q.a.heads[0] + q.a.heads[1] == 0 || q.a.batch == 0 || q.a.tokens == 0) {
    for (int w = 0; kBwd && w < 2; ++w)
      if (a->dweight[w] && cudaMemsetAsync(a->dweight[w], 0, a->head_dim * sizeof(float), st) != cudaSuccess) return PKDA_ERR_LAUNCH;
    return PKDA_OK;
  }
  if (kBwd && (a->dweight[0] || a->dweight[1]) && (!a->workspace || a->workspace_bytes < qk_rotate_bwd_workspace(*a))) return PKDA_ERR_WORKSPACE;
  if (!aligned({a->workspace}, 16)) return PKDA_ERR_ALIGN;
  if (a->dtype == PKDA_BF16) return a->interleaved ? launch_rows<bf16, true, kBwd>(q, st) : launch_rows<bf16, false, kBwd>(q, st);
  return a->interleaved ? launch_rows<float, true, kBwd>(q, st) : launch_rows<float, false, kBwd>(q, st);
}

}  // namespace rotate

int qk_rotate_fwd(const pkda_qk_rotate_args* a, cudaStream_t st) { return rotate::run<false>(a, st); }
int qk_rotate_bwd(const pkda_qk_rotate_args* a, cudaStream_t st) { return rotate::run<true>(a, st); }
size_t qk_rotate_bwd_workspace(const pkda_qk_rotate_args& a) {
  return a.head_dim > 0 ? (size_t)rotate::most_ctas() * 2 * (size_t)a.head_dim * sizeof(float) : 0;
}

}  // namespace pkda

extern "C" {

int pkda_qk_rotate_fwd(const pkda_qk_rotate_args* args, void* cuda_stream) {
  if (!args) return PKDA_ERR_NULL;
  pkda::reset_launch_count();
  return pkda::qk_rotate_fwd(args, static_cast<cudaStream_t>(cuda_stream));
}
size_t pkda_qk_rotate_bwd_workspace_bytes(const pkda_qk_rotate_args* args) { return args ? pkda::qk_rotate_bwd_workspace(*args) : 0; }
int pkda_qk_rotate_bwd(const pkda_qk_rotate_args* args, void* cuda_stream) {
  if (!args) return PKDA_ERR_NULL;
  pkda::reset_launch_count();
  return pkda::qk_rotate_bwd(args, static_cast<cudaStream_t>(cuda_stream));
}
size_t pkda_sizeof_qk_rotate_args(void) { return sizeof(pkda_qk_rotate_args); }

}  // extern "C"
