// Gradients of q, k, g and beta of the chunked gated delta rule, chunk by chunk in parallel, from what the scans have left: the
// states S at a chunk's start and dS' at its end, e and y (gdr_tc.cuh; all split), and the rows q, k, do.
//
//   F1 = do e^T   F2 = y e^T   Cq = s tril(D * F1) diag b   Cm = -tril(diag b D * F2 diag b, -1)
//   dq = Cq k + s exp(G) (S do)       dk = Cq^T q + (Cm + Cm^T) k - exp(G) b (S y) + exp(G_L - G) b (dS' e)
//   dbeta = diag F2
//   dG_i = sum_j R_ij - sum_j R_ji + q_i.(s exp(G_i) S do_i) - k_i.(exp(G_i) b_i S y_i) - c_i,   R = Cq * q k^T + Cm * k k^T,
//   c_i = k_i.(exp(G_L - G_i) b_i dS' e_i),   dg_t = sum_{i >= t} dG_i + sum_i c_i + exp(G_L) <S, dS'>
// A pair's share of dG is one number, added to its row and taken from its column, so the running sum keeps only pairs that
// straddle a token, whatever the gate.
//
// Persistent CTAs, one per SM, over (chunk, key head); the value heads that share the key one after the other, their dq and dk
// summed in tensor memory: the pair products accumulate there, the elementwise warps add the scaled state parts.  Sixteen warps
// do the elementwise work, one issues the products and one the copies; every tile has a barrier of its own, so a tile of the
// next head is asked for, and its products run, while the elementwise work on the head before goes on.  dS' takes the place of S.
// Pair matrices are products with M = 64 (a thread has the same pairs of all four: one decay serves them); the others are
// transposed, channels as lanes, tokens as columns.
//
// 8 x 4,096 tokens of 16 heads: 455 us for 2.28 GB, 0.77 of the copy rate.  What bounds it is the elementwise work of a head, which
// the sixteen warps take phase by phase; the products are in its shadow.
//
// Every wait is bounded, the elementwise warps' for one another as well; a CTA whose wait gives up sets the status word.
#include "gdr_tc.cuh"

namespace pkda {
namespace gdr {

namespace grad {
constexpr int oX = 0;                         // S, then dS': hi and lo, each [16 key octets][128 v][8]
constexpr int oDo = 65536;                    // 2 blocks [64 tok][64 v]
constexpr int oY = oDo + 16384;               // hi, lo: [8 token octets][128 v][8]
constexpr int oE = oY + 32768;                // the same
constexpr int oQ = oE + 32768;                // 2 blocks [64 tok][64 k]
constexpr int oK = oQ + 16384;
constexpr int oCq = oK + 16384, oCm = oCq + 16384;  // hi, lo: [64 i][64 j]
constexpr int oScal = oCm + 16384;            // kScalars fp32, of two heads in turn
constexpr int kScalPitch = kScalars * 4;
// Sums of two heads in turn: f32 [4][64] of rows, of columns and of the state parts, [16][2] carried sums and <S, dS'>.
constexpr int oSums = oScal + 2 * kScalPitch, kSumsPitch = 3 * 1024 + 128;
constexpr int oBar = oSums + 2 * kSumsPitch;
constexpr int kSmem = oBar + 256 + 1024;
constexpr int kThreads = 640;                 // 16 elementwise warps, TMA, products (and two that make up the warpgroup)
constexpr int kWarps = 16;
constexpr int kRegs = 104, kRestRegs = 64;    // 512 x 104 + 128 x 64 = the 640 x 96 of the launch
static_assert(kSmem <= 232448 && oScal % 1024 == 0 && oBar % 8 == 0, "shared memory of one SM");
constexpr uint32_t cQK = 0, cKK = 64, cF1 = 128, cF2 = 192, cSQ = 256, cSY = 320, cDQ = 384, cDK = 448, kCols = 512;
constexpr uint32_t cDE = cF1;                 // (once the pairs have been read)
enum {
  bDoY, bS, bE, bQK, bD, bSc, bSc1,            // tiles have landed (bSc: scalars of even heads, bSc1: of odd ones)
  eDoY, eX, eX2, eE, eQK, eSc, eSc1,           // tiles are free again (eX: S is used up, eX2: dS' is)
  mState, mPairs, mD, mGrad,                   // products are done
  rC,                                          // Cq and Cm stand, F1 and F2 have been read
  rState,                                      // the state parts are in dq and dk, every accumulator has been read
  rSums,                                       // a head's sums stand, and those of the head before have been read
  bCount
};
}  // namespace grad

struct GradParams {
  Params p;
  ChunkBuffers b;
  GradBuffers g;
  bf16 *dq, *dk;
  void* dbeta;
  float* dg;
  Part part;
};

// 16 rows of an accumulator with M = 64, 16 columns, as mma.sync fragments (tmem_ld_rows).
__device__ __forceinline__ void load_rows16(uint32_t taddr, float (&v)[8]) {
  uint32_t* r = reinterpret_cast<uint32_t*>(v);
  asm volatile("tcgen05.ld.sync.aligned.16x256b.x2.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
               : "r"(taddr));
}

__device__ __forceinline__ uint32_t lds_u16(uint32_t addr) {
  unsigned short v;
  asm volatile("ld.shared.u16 %0, [%1];" : "=h"(v) : "r"(addr));
  return v;
}

template <bool kPart>  // (with the division that a part needs the whole takes 475 us, without it 455)
__global__ void __launch_bounds__(grad::kThreads, 1)
gdr_grad_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_do,
                const GradParams a) {
  if (!kPart || !a.part.beside) wait_prerequisites();
  using namespace grad;
  extern __shared__ unsigned char smem_raw[];
  const Params& p = a.p;
  const int H = p.geo.heads, HK = p.key_heads, group = p.group;
  const int tid = threadIdx.x, warp = (int)tc::uniform(tid >> 5), lane = tid & 31;
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  unsigned char* tiles = smem_raw + (base - smem_u32(smem_raw));
  const uint32_t bars = base + oBar, slot = bars + 8 * bCount;
  auto bar = [&](int b) { return bars + 8 * b; };
  if (warp == 0) tc::tmem_alloc(slot, kCols);
  if (tid == 32) {
    for (int b : {(int)bDoY, (int)bS, (int)bE, (int)bQK, (int)bD, (int)bSc, (int)bSc1, (int)eDoY, (int)eX, (int)eE, (int)mState,
                  (int)mPairs, (int)mD, (int)mGrad})
      tc::mbar_init(bar(b), 1);
    for (int b : {(int)eX2, (int)eQK}) tc::mbar_init(bar(b), 1 + kWarps);  // products, and who reads by itself
    for (int b : {(int)eSc, (int)eSc1, (int)rC, (int)rState, (int)rSums}) tc::mbar_init(bar(b), kWarps);
    tc::fence_barrier_init();
  }
  tc::tc_fence_before();
  __syncthreads();
  launch_dependents();
  tc::tc_fence_after();
  const uint32_t tmem = tc::uniform(*reinterpret_cast<volatile uint32_t*>(tiles + oBar + 8 * bCount));
  bool ok = true;
  auto wait = [&](int b, int phase) { ok = __all_sync(0xffffffffu, ok && tc::mbar_wait(bar(b), phase & 1)); };
  auto arrive = [&](int b) {
    __syncwarp();
    if (lane == 0) mbar_arrive(bar(b));
  };
  const int items = (kPart ? part_chunks(p.geo, a.part) : p.geo.total_chunks) * HK;

  if (warp < kWarps) {
    tc::regs_up<kRegs>();
    // ------------------------------------------------------------------------------------------ elementwise
    const int q = warp & 3, cg = warp >> 2, ch = 32 * q + lane;
    const uint32_t cols = tmem + ((uint32_t)(32 * q) << 16) + 16 * cg;  // this warp's lanes, its 16 columns of an accumulator
    // Channel ch of token 16 cg + t in q (k: oK - oQ further): in the swizzled tile its 16-byte piece moves with t % 8.
    const uint32_t row0 = base + oQ + (ch >> 6) * 8192 + 16 * cg * 128 + (ch & 7) * 2, piece = (ch & 63) >> 3;
    int u = 0, it = 0;  // heads and (chunk, key head) items so far
    for (int item = blockIdx.x; item < items && ok; item += gridDim.x) {
      const int x = item / HK, hk = item - x * HK, chunk = kPart ? part_chunk(p.geo, a.part, x) : x;
      int n, tok0, valid;
      if (!chunk_lookup(p.geo, chunk, n, tok0, valid)) break;  // (behind the last chunk: so are all further items)
      for (int g = 0; g < group; ++g, ++u) {
        const int h = hk * group + g;
        const float* sc = reinterpret_cast<const float*>(tiles + oScal + (u & 1) * kScalPitch);
        float* sRow = reinterpret_cast<float*>(tiles + oSums + (u & 1) * kSumsPitch);
        float *sCol = sRow + 256, *sZ = sRow + 512, *sSum = sRow + 768;
        // ---- pairs: rows r0, r0 + 8, columns c0, c0 + 1, c0 + 8, c0 + 9
        wait(bSc + (u & 1), u >> 1);
        wait(mPairs, u);
        if (!ok) break;
        tc::tc_fence_after();
        {
          const int r0 = 16 * q + (lane >> 2), c0 = 16 * cg + 2 * (lane & 3);
          float row[2] = {0.f, 0.f}, col[4] = {0.f, 0.f, 0.f, 0.f};
          if (cg <= q) {  // (a block above the diagonal has no pairs)
            float qk[8], kk[8], f1[8], f2[8];
            load_rows16(cols + cQK, qk);
            load_rows16(cols + cKK, kk);
            load_rows16(cols + cF1, f1);
            load_rows16(cols + cF2, f2);
            tc::tmem_ld_wait();
#pragma unroll
            for (int m = 0; m < 8; m += 2) {  // two neighbouring columns of a row
              const int i = r0 + (m & 2 ? 8 : 0), j0 = c0 + (m & 4 ? 8 : 0);
              const float gi = sc[256 + i], gil = sc[320 + i], bi = sc[64 + i];
              const float2 gj = *reinterpret_cast<const float2*>(sc + 256 + j0), gjl = *reinterpret_cast<const float2*>(sc + 320 + j0),
                           bj = *reinterpret_cast<const float2*>(sc + 64 + j0);
              float cq[2], cm[2];
#pragma unroll
              for (int d = 0; d < 2; ++d) {
                const int j = j0 + d, x = m + d;
                const float b = d ? bj.y : bj.x, w = decay_between(gi, gil, d ? gj.y : gj.x, d ? gjl.y : gjl.x) * b;
                const bool in = i < valid;  // (rows past the end: do is zero there, what the decay is does not matter)
                cq[d] = in && i >= j ? p.scale * w * f1[x] : 0.f;
                cm[d] = in && i > j ? -bi * w * f2[x] : 0.f;
                if (in && i == j) store_dbeta<bf16>(p, a.dbeta, (size_t)(tok0 + i) * H + h, f2[x]);
                const float r = in && i > j ? cq[d] * qk[x] + cm[d] * kk[x] : 0.f;
                row[m & 2 ? 1 : 0] += r;
                col[(m & 4 ? 2 : 0) + d] += r;
              }
              const uint32_t at = i * 128 + (((j0 >> 3) ^ (i & 7)) << 4) + (j0 & 7) * 2;
              uint32_t hi, lo;
              split2(cq[0], cq[1], hi, lo);
              *reinterpret_cast<uint32_t*>(tiles + oCq + at) = hi;
              *reinterpret_cast<uint32_t*>(tiles + oCq + 8192 + at) = lo;
              split2(cm[0], cm[1], hi, lo);
              *reinterpret_cast<uint32_t*>(tiles + oCm + at) = hi;
              *reinterpret_cast<uint32_t*>(tiles + oCm + 8192 + at) = lo;
            }
          } else if (u == 0) {  // zeros there, once
#pragma unroll
            for (int m = 0; m < 8; m += 2) {
              const int i = r0 + (m & 2 ? 8 : 0), j0 = c0 + (m & 4 ? 8 : 0);
              const uint32_t at = i * 128 + (((j0 >> 3) ^ (i & 7)) << 4) + (j0 & 7) * 2;
#pragma unroll
              for (int part = 0; part < 4; ++part) *reinterpret_cast<uint32_t*>(tiles + oCq + 8192 * part + at) = 0u;
            }
          }
          tc::fence_proxy_async();
          tc::tc_fence_before();
          arrive(rC);
#pragma unroll
          for (int d = 0; d < 2; ++d) {
            row[d] += __shfl_xor_sync(0xffffffffu, row[d], 1);
            row[d] += __shfl_xor_sync(0xffffffffu, row[d], 2);
            if ((lane & 3) == 0) sRow[cg * 64 + r0 + 8 * d] = row[d];
          }
#pragma unroll
          for (int d = 0; d < 4; ++d) {
#pragma unroll
            for (int o = 4; o < 32; o <<= 1) col[d] += __shfl_xor_sync(0xffffffffu, col[d], o);
            if (lane < 4) sCol[q * 64 + 16 * cg + 2 * lane + (d & 1) + (d & 2 ? 8 : 0)] = col[d];
          }
        }
        // ---- channel ch of q and k, tokens 16 cg + t, two to a word (then q and k may go)
        wait(bQK, it);
        if (!ok) break;
        uint32_t qv[8], kv[8];
        {
          uint32_t base_t[8];  // (by address: loads that nothing holds up)
#pragma unroll
          for (int t = 0; t < 8; ++t) base_t[t] = row0 + t * 128 + ((piece ^ t) << 4);
#pragma unroll
          for (int t = 0; t < 8; ++t) {
            const uint32_t e = base_t[(2 * t) & 7] + (t >> 2) * 1024, o = base_t[(2 * t + 1) & 7] + (t >> 2) * 1024;
            qv[t] = __byte_perm(lds_u16(e), lds_u16(o), 0x5410);
            kv[t] = __byte_perm(lds_u16(e + (oK - oQ)), lds_u16(o + (oK - oQ)), 0x5410);
          }
          if (g + 1 == group) {
            uint32_t seen = 0;
#pragma unroll
            for (int t = 0; t < 8; ++t) seen ^= qv[t] ^ kv[t];
            arrive_behind_loads(bar(eQK), seen);
          }
          if (valid < kChunk) {  // rows past the end are another sequence's
#pragma unroll
            for (int t = 0; t < 8; ++t) {
              const uint32_t m = (16 * cg + 2 * t < valid ? 0xffffu : 0u) | (16 * cg + 2 * t + 1 < valid ? 0xffff0000u : 0u);
              qv[t] &= m;
              kv[t] &= m;
            }
          }
        }
        // ---- <S, dS'>: this thread's 32 elements of S come once more, from L2, which they have just passed (kept in registers
        // since they stood in shared memory they would cost what the pairs need; not from the first level: chunk_scalars)
        uint4 sh[4], sl[4];
        {
          const uint4* s4 = reinterpret_cast<const uint4*>(a.b.h + ((size_t)chunk * H + h) * 2 * kW * kW) + tid;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            sh[j] = __ldcg(s4 + j * 512);
            sl[j] = __ldcg(s4 + 2048 + j * 512);
          }
        }
        wait(bD, u);
        if (!ok) break;
        float2 dot2 = f2(0.f, 0.f);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint4 dh = *reinterpret_cast<const uint4*>(tiles + oX + (j * 512 + tid) * 16);
          const uint4 dl = *reinterpret_cast<const uint4*>(tiles + oX + 32768 + (j * 512 + tid) * 16);
          const uint32_t a0[4] = {sh[j].x, sh[j].y, sh[j].z, sh[j].w}, a1[4] = {sl[j].x, sl[j].y, sl[j].z, sl[j].w},
                         b0[4] = {dh.x, dh.y, dh.z, dh.w}, b1[4] = {dl.x, dl.y, dl.z, dl.w};
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const float2 s0 = unpack_bf16(a0[c]), s1 = unpack_bf16(a1[c]), d0 = unpack_bf16(b0[c]), d1 = unpack_bf16(b1[c]);
            dot2 = fma2(add2(s0, s1), add2(d0, d1), dot2);
          }
        }
        float dot = dot2.x + dot2.y;
        arrive_behind_loads(bar(eX2), __float_as_uint(dot));
        // ---- what the states give, onto the pair parts
        wait(mState, u);
        wait(mGrad, u);
        wait(mD, u);
        if (!ok) break;
        tc::tc_fence_after();
        float z[16], carry = 0.f;
#pragma unroll
        for (int half = 0; half < 16; half += 8) {
          float x[8], y[8], e[8], dq[8], dk[8];
          tc::tmem_ld8(cols + cSQ + half, x);
          tc::tmem_ld8(cols + cSY + half, y);
          tc::tmem_ld8(cols + cDE + half, e);
          tc::tmem_ld8(cols + cDQ + half, dq);
          tc::tmem_ld8(cols + cDK + half, dk);
          tc::tmem_ld_wait();
#pragma unroll
          for (int t = 0; t < 8; t += 2) {  // two tokens at a time
            const float* s0 = sc + 16 * cg + half + t;
            const float2 gam = *reinterpret_cast<const float2*>(s0), bet = *reinterpret_cast<const float2*>(s0 + 64),
                         kap = *reinterpret_cast<const float2*>(s0 + 128);
            const float2 qq = unpack_bf16(qv[(half + t) / 2]), kk = unpack_bf16(kv[(half + t) / 2]);
            const float2 a0 = mul2(mul2(gam, f2(p.scale, p.scale)), f2(x[t], x[t + 1])), a1 = mul2(mul2(gam, bet), f2(-y[t], -y[t + 1])),
                         a2 = mul2(kap, f2(e[t], e[t + 1]));
            const float2 nq = add2(f2(dq[t], dq[t + 1]), a0), nk = add2(f2(dk[t], dk[t + 1]), add2(a1, a2));
            dq[t] = nq.x; dq[t + 1] = nq.y;
            dk[t] = nk.x; dk[t + 1] = nk.y;
            const float2 w = mul2(kk, a2), zz = fma2(qq, a0, fma2(kk, a1, f2(-w.x, -w.y)));
            z[half + t] = zz.x;
            z[half + t + 1] = zz.y;
            carry += w.x + w.y;
          }
          if (g + 1 < group) {
            tc::tmem_st8(cols + cDQ + half, dq);
            tc::tmem_st8(cols + cDK + half, dk);
          } else {
            const size_t at = ((size_t)(tok0 + 16 * cg + half) * HK + hk) * kW + ch, step = (size_t)HK * kW;
#pragma unroll
            for (int t = 0; t < 8; ++t) {
              if (16 * cg + half + t < valid) {
                a.dq[at + t * step] = __float2bfloat16(dq[t]);
                a.dk[at + t * step] = __float2bfloat16(dk[t]);
              }
            }
          }
        }
        tc::tmem_st_wait();
        tc::tc_fence_before();
        arrive(rState);
        // sums over the lanes: z is folded by halves (lane bits 4..1 choose a token), the two sums follow plainly
#pragma unroll
        for (int w = 16; w > 1; w >>= 1) {
          const int half = w / 2;
          const bool up = lane & w;
#pragma unroll
          for (int t = 0; t < half; ++t) {
            const float give = up ? z[t] : z[t + half], keep = up ? z[t + half] : z[t];
            z[t] = keep + __shfl_xor_sync(0xffffffffu, give, w);
          }
        }
        z[0] += __shfl_xor_sync(0xffffffffu, z[0], 1);
        if (!(lane & 1)) sZ[q * 64 + 16 * cg + (lane >> 1)] = z[0];
#pragma unroll
        for (int o = 16; o; o >>= 1) {
          carry += __shfl_xor_sync(0xffffffffu, carry, o);
          dot += __shfl_xor_sync(0xffffffffu, dot, o);
        }
        if (lane == 0) {
          sSum[2 * warp] = carry;
          sSum[2 * warp + 1] = dot;
        }
        arrive(rSums);  // (a named barrier has no limit: a warp that has given up would hold the others there)
        wait(rSums, u);
        if (!ok) break;
        uint32_t seen = 0;
        if (warp == 0) {  // reverse cumulative sum: lane l has tokens 2 l and 2 l + 1
          float x[2], run = 0.f, end = 0.f, whole = 0.f;
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const int t = 2 * lane + j;
            x[j] = (sRow[t] + sRow[64 + t] + sRow[128 + t] + sRow[192 + t]) - (sCol[t] + sCol[64 + t] + sCol[128 + t] + sCol[192 + t]) +
                   (sZ[t] + sZ[64 + t] + sZ[128 + t] + sZ[192 + t]);
          }
          run = x[0] + x[1];
          end = lane < 16 ? sSum[2 * lane] : 0.f;
          whole = lane < 16 ? sSum[2 * lane + 1] : 0.f;
#pragma unroll
          for (int o = 16; o; o >>= 1) {
            end += __shfl_xor_sync(0xffffffffu, end, o);
            whole += __shfl_xor_sync(0xffffffffu, whole, o);
          }
          end += sc[63] * whole;  // exp(G_L)
#pragma unroll
          for (int o = 1; o < 32; o <<= 1) {
            const float w = __shfl_down_sync(0xffffffffu, run, o);
            if (lane + o < 32) run += w;
          }
          float* out = a.dg + (size_t)tok0 * H + h;
          if (2 * lane < valid) out[(size_t)(2 * lane) * H] = run + end;
          if (2 * lane + 1 < valid) out[(size_t)(2 * lane + 1) * H] = run - x[0] + end;
          seen = __float_as_uint(end);
        }
        arrive_behind_loads(bar(eSc + (u & 1)), seen);  // (the other scalars are in sums that have been exchanged)
      }
      if (!ok) break;
      ++it;
    }
    if (!ok && lane == 0) atomicExch(a.b.status, 1);
  } else {
    tc::regs_down<kRestRegs>();
    if (warp == kWarps) {
      // ---------------------------------------------------------------------------------------- TMA
      if (lane == 0) {
        int u = 0, it = 0;
        auto free_again = [&](int b, int uses) { ok = ok && (uses == 0 || tc::mbar_wait(bar(b), (uses - 1) & 1)); };
        for (int item = blockIdx.x; item < items && ok; item += gridDim.x, ++it) {
          const int x = item / HK, hk = item - x * HK, chunk = kPart ? part_chunk(p.geo, a.part, x) : x;
          int n, tok0, valid;
          if (!chunk_lookup(p.geo, chunk, n, tok0, valid)) break;
          for (int g = 0; g < group && ok; ++g, ++u) {
            const int h = hk * group + g;
            const size_t ci = (size_t)chunk * H + h;
            free_again(eSc + (u & 1), u >> 1);
            if (!ok) break;
            tc::mbar_expect_tx(bar(bSc + (u & 1)), kScalars * 4);
            tc::bulk_load(base + oScal + (u & 1) * kScalPitch, a.b.scal + ci * kScalars, kScalars * 4, bar(bSc + (u & 1)));
            free_again(eDoY, u);
            if (!ok) break;
            tc::mbar_expect_tx(bar(bDoY), 49152);
#pragma unroll
            for (int b = 0; b < 2; ++b) tc::tma_load_3d(base + oDo + 8192 * b, &tm_do, bar(bDoY), 64 * b, h, tok0);
            tc::bulk_load(base + oY, a.g.y + ci * 2 * kW * 64, 32768, bar(bDoY));
            if (g == 0) {
              free_again(eQK, it);
              if (!ok) break;
              tc::mbar_expect_tx(bar(bQK), 32768);
#pragma unroll
              for (int b = 0; b < 2; ++b) {
                tc::tma_load_3d(base + oQ + 8192 * b, &tm_q, bar(bQK), 64 * b, hk, tok0);
                tc::tma_load_3d(base + oK + 8192 * b, &tm_k, bar(bQK), 64 * b, hk, tok0);
              }
            }
            free_again(eE, u);
            if (!ok) break;
            tc::mbar_expect_tx(bar(bE), 32768);
            tc::bulk_load(base + oE, a.b.e + ci * 2 * kW * 64, 32768, bar(bE));
            free_again(eX2, u);
            if (!ok) break;
            tc::mbar_expect_tx(bar(bS), 65536);
            tc::bulk_load(base + oX, a.b.h + ci * 2 * kW * kW, 65536, bar(bS));
            free_again(eX, u + 1);  // S of this head is used up
            if (!ok) break;
            tc::mbar_expect_tx(bar(bD), 65536);
            tc::bulk_load(base + oX, a.g.dh + ci * 2 * kW * kW, 65536, bar(bD));
          }
        }
        if (!ok) {
          atomicExch(a.b.status, 1);
          // copies in flight have to land before the CTA's shared memory goes to another: the last phase of each tile's barrier
          for (int b : {(int)bDoY, (int)bS, (int)bE, (int)bD, (int)bSc, (int)bSc1})
            if (u > 0) tc::mbar_wait(bar(b), 0), tc::mbar_wait(bar(b), 1);
          if (u > 0) tc::mbar_wait(bar(bQK), 0), tc::mbar_wait(bar(bQK), 1);
        }
      }
    } else if (warp == kWarps + 1) {
      // ---------------------------------------------------------------------------------------- the products
      constexpr uint32_t s_do = tc::idesc_bf16(128, 64, true, false), s_y = tc::idesc_bf16(128, 64, true, true),
                         p_kk = tc::idesc_bf16(64, 64, false, false), p_de = tc::idesc_bf16(64, 64, false, true),
                         p_ye = tc::idesc_bf16(64, 64, true, true);
      int u = 0, it = 0;
      for (int item = blockIdx.x; item < items && ok; item += gridDim.x, ++it) {
        const int chunk = kPart ? part_chunk(p.geo, a.part, item / HK) : item / HK;
        int n, tok0, valid;
        if (!chunk_lookup(p.geo, chunk, n, tok0, valid)) break;
        for (int g = 0; g < group && ok; ++g, ++u) {
          uint32_t b0 = base;
          asm volatile("" : "+r"(b0));  // (else two hundred descriptors are formed in front of the loop and spilled)
          b0 = tc::uniform(b0);
          if (g == 0) {
            wait(bQK, it);
            if (!ok) break;
            if (valid < kChunk) {
              zero_rows(tiles + oQ, 8192, valid);
              zero_rows(tiles + oK, 8192, valid);
            }
          }
          wait(bDoY, u);
          if (!ok) break;
          if (valid < kChunk) {
            zero_rows(tiles + oDo, 8192, valid);
            tc::fence_proxy_async();
            __syncwarp();
          }
          wait(bE, u);
          if (!ok) break;
          if (tc::elect_one()) {  // (the pairs of the head before have been read: rC)
#pragma unroll
            for (int kk = 0; kk < 8; ++kk) {
              const uint32_t k = b0 + oK + (kk >> 2) * 8192 + (kk & 3) * 32;
              tc::umma_bf16(tmem + cQK, tc::desc_kmajor(b0 + oQ + (kk >> 2) * 8192 + (kk & 3) * 32), tc::desc_kmajor(k), p_kk, kk > 0);
              tc::umma_bf16(tmem + cKK, tc::desc_kmajor(k), tc::desc_kmajor(k), p_kk, kk > 0);
            }
#pragma unroll
            for (int kk = 0; kk < 24; ++kk)  // y e^T: hi hi, hi lo, lo hi
              tc::umma_bf16(tmem + cF2, octet_desc(b0 + oY + (kk >> 3 == 2 ? 16384 : 0), kk & 7),
                            octet_desc(b0 + oE + (kk >> 3 == 1 ? 16384 : 0), kk & 7), p_ye, kk > 0);
          }
          __syncwarp();
          if (u > 0) wait(rState, u - 1);
          if (!ok) break;
          tc::tc_fence_after();
          if (tc::elect_one()) {
#pragma unroll
            for (int kk = 0; kk < 16; ++kk)  // do e^T
              tc::umma_bf16(tmem + cF1, tc::desc_kmajor(b0 + oDo + ((kk >> 2) & 1) * 8192 + (kk & 3) * 32),
                            octet_desc(b0 + oE + (kk >> 3) * 16384, kk & 7), p_de, kk > 0);
            tc::umma_commit(bar(mPairs));
          }
          __syncwarp();
          wait(bS, u);
          if (!ok) break;
          if (tc::elect_one()) {
#pragma unroll
            for (int kk = 0; kk < 16; ++kk)  // S do^T: S hi, S lo
              tc::umma_bf16(tmem + cSQ, octet_desc(b0 + oX + (kk >> 3) * 32768, kk & 7),
                            tc::desc_kmajor(b0 + oDo + ((kk >> 2) & 1) * 8192 + (kk & 3) * 32), s_do, kk > 0);
#pragma unroll
            for (int kk = 0; kk < 24; ++kk)  // S y^T: hi hi, lo hi, hi lo
              tc::umma_bf16(tmem + cSY, octet_desc(b0 + oX + (kk >> 3 == 1 ? 32768 : 0), kk & 7),
                            octet_desc(b0 + oY + (kk >> 3 == 2 ? 16384 : 0), kk & 7), s_y, kk > 0);
            tc::umma_commit(bar(mState));
            tc::umma_commit(bar(eX));
            tc::umma_commit(bar(eDoY));
          }
          __syncwarp();
          wait(rC, u);
          if (!ok) break;
          tc::tc_fence_after();
          if (tc::elect_one()) {  // every matrix hi, then lo; onto the sums of the heads before
#pragma unroll
            for (int kk = 0; kk < 8; ++kk)
              tc::umma_bf16(tmem + cDQ, tc::desc_mnmajor(b0 + oK + (kk & 3) * 2048, 8192),
                            tc::desc_kmajor(b0 + oCq + (kk >> 2) * 8192 + (kk & 3) * 32), s_do, kk > 0 || g > 0);
#pragma unroll
            for (int kk = 0; kk < 8; ++kk)
              tc::umma_bf16(tmem + cDK, tc::desc_mnmajor(b0 + oQ + (kk & 3) * 2048, 8192),
                            tc::desc_mnmajor(b0 + oCq + (kk >> 2) * 8192 + (kk & 3) * 2048, 8192), s_y, kk > 0 || g > 0);
#pragma unroll
            for (int kk = 0; kk < 8; ++kk)
              tc::umma_bf16(tmem + cDK, tc::desc_mnmajor(b0 + oK + (kk & 3) * 2048, 8192),
                            tc::desc_kmajor(b0 + oCm + (kk >> 2) * 8192 + (kk & 3) * 32), s_do, 1);
#pragma unroll
            for (int kk = 0; kk < 8; ++kk)
              tc::umma_bf16(tmem + cDK, tc::desc_mnmajor(b0 + oK + (kk & 3) * 2048, 8192),
                            tc::desc_mnmajor(b0 + oCm + (kk >> 2) * 8192 + (kk & 3) * 2048, 8192), s_y, 1);
            tc::umma_commit(bar(mGrad));
            if (g + 1 == group) tc::umma_commit(bar(eQK));
          }
          __syncwarp();
          wait(bD, u);
          if (!ok) break;
          if (tc::elect_one()) {
#pragma unroll
            for (int kk = 0; kk < 24; ++kk)  // dS' e^T, where do e^T was
              tc::umma_bf16(tmem + cDE, octet_desc(b0 + oX + (kk >> 3 == 1 ? 32768 : 0), kk & 7),
                            octet_desc(b0 + oE + (kk >> 3 == 2 ? 16384 : 0), kk & 7), s_y, kk > 0);
            tc::umma_commit(bar(mD));
            tc::umma_commit(bar(eX2));
            tc::umma_commit(bar(eE));
          }
          __syncwarp();
        }
      }
      if (!ok && lane == 0) atomicExch(a.b.status, 1);
    }
  }
  tc::tc_fence_before();
  __syncthreads();
  if (warp == 0) tc::tmem_dealloc(tmem, kCols);
  if (kPart && a.part.beside && blockIdx.x == 0) wait_prerequisites();
  // If a kernel of the backward gave up (this CTA included), the first row of this CTA's gradients becomes NaN.
  if (warp == 1 && (int)blockIdx.x < items && *reinterpret_cast<volatile int*>(a.b.status) != 0) {
    const int x = blockIdx.x / HK, hk = blockIdx.x - x * HK;
    int n, tok0, valid;
    if (chunk_lookup(p.geo, kPart ? part_chunk(p.geo, a.part, x) : x, n, tok0, valid)) {
      const size_t row = ((size_t)tok0 * HK + hk) * kW, heads = (size_t)tok0 * H + hk * group;
      mark_failed(a.dq + row, kW);
      mark_failed(a.dk + row, kW);
      mark_failed(a.dg + heads, group);
      if (p.beta32) mark_failed(static_cast<float*>(a.dbeta) + heads, group);
      else mark_failed(static_cast<bf16*>(a.dbeta) + heads, group);
    }
  }
}

int launch_grad(const Params& p, const ChunkBuffers& b, const GradBuffers& g, const Part& part, const bf16* d_o, bf16* dq, bf16* dk, float* dg,
                void* dbeta, cudaStream_t st) {
  const int tok = p.geo.total_tokens;
  CUtensorMap tm_q, tm_k, tm_do;
  if (!map_rows(&tm_q, p.q, p.key_heads, tok) || !map_rows(&tm_k, p.k, p.key_heads, tok) || !map_rows(&tm_do, d_o, p.geo.heads, tok))
    return PKDA_ERR_LAUNCH;
  GradParams a;
  a.p = p; a.b = b; a.g = g; a.part = part; a.dq = dq; a.dk = dk; a.dg = dg; a.dbeta = dbeta;
  const auto kernel = part.c1 ? gdr_grad_kernel<true> : gdr_grad_kernel<false>;
  if (!ensure_dynamic_smem(kernel, grad::kSmem)) return PKDA_ERR_LAUNCH;
  // (beside a scan: on the SMs that it leaves)
  const int work = part_chunks(p.geo, part) * p.key_heads, sms = sm_count() - (part.beside ? p.geo.n_seqs * p.geo.heads : 0);
  begin_stage(kStageGdrChunkGrad, st);
  const int rc = launch_kernel(kernel, work < sms ? work : sms, grad::kThreads, grad::kSmem, st, tm_q, tm_k, tm_do, a);
  end_stage(st);
  return rc;
}

}  // namespace gdr
}  // namespace pkda
