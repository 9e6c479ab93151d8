// Pair matrices of the chunked gated delta rule: per (chunk, key head) the products k k^T and q k^T once, then for each of
// the value heads that share the key P, N = (I + M diag b)^-1 M and from it T (and T2), see gdr_tc.cuh.
//
// One CTA of 256 threads per (chunk, key head), four to an SM.  [k; q] k^T is one tcgen05 product (M = 128, N = 64, K = 128) of the
// rows as TMA brings them; a thread reads back half a row, k rows for M, q rows for P, and applies the decays.  N is solved in fp32 on the
// CUDA cores (its terms cancel where keys are alike, which bf16 or TF32 products would not survive): the eight diagonal blocks
// of 8 by substitution, a warp each, then three levels of
//   N21 = X - N22 (b2 X),   X = M21 - M21 (b1 N11)
// with a thread per column and 1, 2 or 4 rows.  What bounds it is the chain of these phases: 198 us for 8 x 4,096 tokens of
// 16 heads, whose 0.7 GB would take 104 at the copy rate (blocks of 16 by substitution, 128 threads an item: 219 us).  Four CTAs on an
// SM leave 64 registers a thread, which spills two to ten words around the loop over the heads.
#include "gdr_tc.cuh"

namespace pkda {
namespace gdr {

namespace pairs {
constexpr int kThreads = 256;
constexpr int kLd = 68;                     // row stride of the fp32 matrices
constexpr int oA = 0;                       // 2 blocks [128 rows][64 ch]: k rows, q rows
constexpr int oM = oA;                      // f32 [64][68], where the operands were
constexpr int oN = 32768;                   // f32 [64][68]
constexpr int oY = oM + 64 * kLd * 4;       // f32 [32][36] right-hand sides of a merge
constexpr int oG = oN + 64 * kLd * 4;       // f32 [64] each: G in units of log 2, hi and lo, and beta; of two heads in turn
constexpr int kScal = 768;
constexpr int oBar = oG + 2 * kScal;
constexpr int kSmem = oBar + 64 + 1024;
constexpr int kTx = 32768;
constexpr int kLdY = 36;
static_assert(oY + 32 * kLdY * 4 <= 32768, "fits in front of N");
static_assert(oN % 16 == 0 && oY % 16 == 0, "float4 rows");
}  // namespace pairs

struct PairParams {
  Params p;
  ChunkBuffers b;
  Part part;
};

// Eight values of a matrix row to their place in the hi part and in the lo part behind it.
__device__ __forceinline__ void store_split(uint4* at, const float (&x)[8]) {
  uint4 hi, lo;
  split2(x[0], x[1], hi.x, lo.x);
  split2(x[2], x[3], hi.y, lo.y);
  split2(x[4], x[5], hi.z, lo.z);
  split2(x[6], x[7], hi.w, lo.w);
  *at = hi;
  at[8 * 64] = lo;
}

template <bool kPart>  // (a part's chunk number is one register too many)
__global__ void __launch_bounds__(pairs::kThreads, 4)
gdr_pairs_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_q, const PairParams a) {
  if (!kPart || !a.part.beside) wait_prerequisites();
  using namespace pairs;
  extern __shared__ unsigned char smem_raw[];
  const Params& p = a.p;
  int n, tok0, valid;
  auto chunk = [&] { return (int)(kPart ? blockIdx.z * p.geo.chunks_per_seq + a.part.c0 + blockIdx.x : blockIdx.x); };
  const bool mine = chunk_lookup(p.geo, chunk(), n, tok0, valid);
  const int hk = blockIdx.y, H = p.geo.heads, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (!mine) return;
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  unsigned char* tiles = smem_raw + (base - smem_u32(smem_raw));
  float* sM = reinterpret_cast<float*>(tiles + oM);
  float* sN = reinterpret_cast<float*>(tiles + oN);
  float* sY = reinterpret_cast<float*>(tiles + oY);
  const uint32_t bar_full = base + oBar, bar_mma = base + oBar + 8, slot = base + oBar + 16;
  if (warp == 0) tc::tmem_alloc(slot, 64);
  if (tid == 32) {
    tc::mbar_init(bar_full, 1);
    tc::mbar_init(bar_mma, 1);
    tc::fence_barrier_init();
    tc::mbar_expect_tx(bar_full, kTx);
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      tc::tma_load_3d(base + oA + b * 16384, &tm_k, bar_full, 64 * b, hk, tok0);
      tc::tma_load_3d(base + oA + b * 16384 + 8192, &tm_q, bar_full, 64 * b, hk, tok0);
    }
  }
  tc::tc_fence_before();
  __syncthreads();
  launch_dependents();
  tc::tc_fence_after();
  const uint32_t tmem = tc::uniform(*reinterpret_cast<volatile uint32_t*>(tiles + oBar + 16));
  // Decays and betas of head g: while the tiles are on their way, or while the head before is written out.
  auto scalars = [&](int g) {
    const int h = hk * p.group + g;
    const size_t at = (size_t)tok0 * H + h;
    float* sG = reinterpret_cast<float*>(tiles + oG + (g & 1) * kScal);
    const double total = chunk_scalars<bf16>(p, at, valid, sG, sG + 64, sG + 128);
    __syncwarp();
    float* out = a.b.scal + ((size_t)chunk() * H + h) * kScalars;
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const int t = lane + 32 * half;
      const float G = sG[t], Gl = sG[64 + t], b = sG[128 + t], rest = exp2f((float)(total - (double)G - (double)Gl));
      out[t] = exp2f(G + Gl);
      out[64 + t] = b;
      out[128 + t] = rest * b;
      out[192 + t] = rest;
      out[256 + t] = G;
      out[320 + t] = Gl;
    }
  };
  if (warp == 7) scalars(0);
  bool ok = tc::mbar_wait(bar_full, 0);
  if (ok && tc::uniform(warp) == 0 && tc::elect_one()) {
    constexpr uint32_t idesc = tc::idesc_bf16(128, 64, false, false);
#pragma unroll
    for (int kk = 0; kk < 8; ++kk) {
      const uint32_t at = base + oA + (kk >> 2) * 16384 + (kk & 3) * 32;
      tc::umma_bf16(tmem, tc::desc_kmajor(at), tc::desc_kmajor(at), idesc, kk > 0);
    }
    tc::umma_commit(bar_mma);
  }
  __syncwarp();
  ok = tc::mbar_wait(bar_mma, 0) && ok;
  if (__syncthreads_or(!ok)) {
    if (tid == 0) atomicExch(a.b.status, 1);
  } else {
    tc::tc_fence_after();
    const int quad = warp & 3, j0 = 32 * (warp >> 2);  // this warp's 32 rows (two of k, two of q) and 32 columns
    float row[32];
    tc::tmem_ld32(tmem + ((uint32_t)(32 * quad) << 16) + j0, row);
    tc::tmem_ld_wait();
    const int i = (32 * quad + lane) & 63;  // token of this thread's row
    for (int g = 0; g < p.group; ++g) {
      const int h = hk * p.group + g;
      const size_t item = (size_t)chunk() * H + h;
      const float* sG = reinterpret_cast<const float*>(tiles + oG + (g & 1) * kScal);
      const float* sB = sG + 128;
      __syncthreads();  // the scalars stand (and the matrices of the head before are done with)
      const float Gi = sG[i], Gli = sG[64 + i];
      auto decay = [&](int j) { return decay_between(Gi, Gli, sG[j], sG[64 + j]); };
      if (quad < 2) {
        float* m = sM + i * kLd + j0;
#pragma unroll
        for (int j = 0; j < 32; j += 4) {
          float x[4];
#pragma unroll
          for (int c = 0; c < 4; ++c) x[c] = j0 + j + c < i && i < valid ? row[j + c] * decay(j0 + j + c) : 0.f;
          *reinterpret_cast<float4*>(m + j) = make_float4(x[0], x[1], x[2], x[3]);
        }
      } else {
        uint4* out = reinterpret_cast<uint4*>(a.b.P + item * 2 * 4096) + 8 * j0 + i;
#pragma unroll
        for (int j = 0; j < 32; j += 8) {
          float x[8];
#pragma unroll
          for (int c = 0; c < 8; ++c) x[c] = j0 + j + c <= i && i < valid ? p.scale * row[j + c] * decay(j0 + j + c) : 0.f;
          store_split(out + 8 * j, x);
        }
      }
      __syncthreads();

      // ---- diagonal blocks of 8, a warp each: lane c has column c (lanes 8.. repeat them and write nothing)
      {
        const int c = lane & 7, o = 8 * warp;
        const float4 b0 = *reinterpret_cast<const float4*>(sB + o), b1 = *reinterpret_cast<const float4*>(sB + o + 4);
        const float b[8] = {b0.x, b0.y, b0.z, b0.w, b1.x, b1.y, b1.z, b1.w};
        float x[8], nb[8];  // column c of the block; beta_l N_lc
#pragma unroll
        for (int r = 0; r < 8; ++r) x[r] = sM[(o + r) * kLd + o + c];
#pragma unroll
        for (int r = 0; r < 8; ++r) {
#pragma unroll
          for (int l4 = 0; l4 < r; l4 += 4) {
            const float4 m = *reinterpret_cast<const float4*>(sM + (o + r) * kLd + o + l4);
            if (l4 < r) x[r] -= m.x * nb[l4];
            if (l4 + 1 < r) x[r] -= m.y * nb[l4 + 1];
            if (l4 + 2 < r) x[r] -= m.z * nb[l4 + 2];
            if (l4 + 3 < r) x[r] -= m.w * nb[l4 + 3];
          }
          // (above the diagonal M is zero, so x is too: no case for r <= c)
          nb[r] = b[r] * x[r];
          if (lane < 8) sN[(o + r) * kLd + o + c] = x[r];
        }
        // zeros right of the odd blocks' left neighbours and of the odd 16-blocks', which the next levels read as part of N11, N22
        if (!(warp & 1) && lane >= 16)
          *reinterpret_cast<float4*>(sN + (o + ((lane - 16) >> 1)) * kLd + o + 8 + (lane & 1) * 4) = make_float4(0.f, 0.f, 0.f, 0.f);
        if (!(warp & 2)) {
          const int r = 32 * (warp >> 2) + 8 * (warp & 1) + (lane >> 2), cc = 32 * (warp >> 2) + 16 + (lane & 3) * 4;
          *reinterpret_cast<float4*>(sN + r * kLd + cc) = make_float4(0.f, 0.f, 0.f, 0.f);
        }
      }
      __syncthreads();
      // ---- 8 -> 16: four pairs of blocks, a thread an element
      {
        const int pr = tid >> 6, c = tid & 7, r = (tid >> 3) & 7, b1 = 16 * pr, b2 = b1 + 8;
        float x = sM[(b2 + r) * kLd + b1 + c];
#pragma unroll
        for (int l = 0; l < 8; l += 4) {
          const float4 m = *reinterpret_cast<const float4*>(sM + (b2 + r) * kLd + b1 + l), b = *reinterpret_cast<const float4*>(sB + b1 + l);
          x -= m.x * (b.x * sN[(b1 + l) * kLd + b1 + c]) + m.y * (b.y * sN[(b1 + l + 1) * kLd + b1 + c]) +
               m.z * (b.z * sN[(b1 + l + 2) * kLd + b1 + c]) + m.w * (b.w * sN[(b1 + l + 3) * kLd + b1 + c]);
        }
        sY[(8 * pr + r) * kLdY + c] = sB[b2 + r] * x;
        __syncthreads();
#pragma unroll
        for (int l = 0; l < 8; l += 4) {
          const float4 m = *reinterpret_cast<const float4*>(sN + (b2 + r) * kLd + b2 + l);
          x -= m.x * sY[(8 * pr + l) * kLdY + c] + m.y * sY[(8 * pr + l + 1) * kLdY + c] + m.z * sY[(8 * pr + l + 2) * kLdY + c] +
               m.w * sY[(8 * pr + l + 3) * kLdY + c];
        }
        sN[(b2 + r) * kLd + b1 + c] = x;
      }
      __syncthreads();
      // ---- 16 -> 32: two pairs of blocks, 128 threads each, a column and two rows a thread
      {
        const int pr = tid >> 7, c = tid & 15, r0 = ((tid & 127) >> 4) * 2, b1 = 32 * pr, b2 = b1 + 16;
        float x[2];
#pragma unroll
        for (int r = 0; r < 2; ++r) x[r] = sM[(b2 + r0 + r) * kLd + b1 + c];
#pragma unroll
        for (int l = 0; l < 16; l += 4) {
          const float4 b = *reinterpret_cast<const float4*>(sB + b1 + l);
          const float nb[4] = {b.x * sN[(b1 + l) * kLd + b1 + c], b.y * sN[(b1 + l + 1) * kLd + b1 + c], b.z * sN[(b1 + l + 2) * kLd + b1 + c],
                               b.w * sN[(b1 + l + 3) * kLd + b1 + c]};
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            const float4 m = *reinterpret_cast<const float4*>(sM + (b2 + r0 + r) * kLd + b1 + l);
            x[r] -= m.x * nb[0] + m.y * nb[1] + m.z * nb[2] + m.w * nb[3];
          }
        }
#pragma unroll
        for (int r = 0; r < 2; ++r) sY[(16 * pr + r0 + r) * kLdY + c] = sB[b2 + r0 + r] * x[r];
        __syncthreads();
#pragma unroll
        for (int l = 0; l < 16; l += 4) {
          float y[4];
#pragma unroll
          for (int d = 0; d < 4; ++d) y[d] = sY[(16 * pr + l + d) * kLdY + c];
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            const float4 m = *reinterpret_cast<const float4*>(sN + (b2 + r0 + r) * kLd + b2 + l);
            x[r] -= m.x * y[0] + m.y * y[1] + m.z * y[2] + m.w * y[3];
          }
        }
#pragma unroll
        for (int r = 0; r < 2; ++r) sN[(b2 + r0 + r) * kLd + b1 + c] = x[r];
      }
      __syncthreads();
      // ---- 32 -> 64: lane = column, four rows a warp
      {
        const int c = lane, r0 = 32 + 4 * warp;
        float x[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) x[r] = sM[(r0 + r) * kLd + c];
#pragma unroll 4
        for (int l = 0; l < 32; l += 4) {
          const float4 b = *reinterpret_cast<const float4*>(sB + l);
          const float nb[4] = {b.x * sN[l * kLd + c], b.y * sN[(l + 1) * kLd + c], b.z * sN[(l + 2) * kLd + c], b.w * sN[(l + 3) * kLd + c]};
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const float4 m = *reinterpret_cast<const float4*>(sM + (r0 + r) * kLd + l);
            x[r] -= m.x * nb[0] + m.y * nb[1] + m.z * nb[2] + m.w * nb[3];
          }
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) sY[(4 * warp + r) * kLdY + c] = sB[r0 + r] * x[r];
        __syncthreads();
#pragma unroll 4
        for (int l = 0; l < 4 * warp + 4; l += 4) {  // (row r of N22 ends in front of its diagonal)
          float y[4];
#pragma unroll
          for (int d = 0; d < 4; ++d) y[d] = sY[(l + d) * kLdY + c];
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const float4 m = *reinterpret_cast<const float4*>(sN + (r0 + r) * kLd + 32 + l);
            x[r] -= m.x * y[0] + m.y * y[1] + m.z * y[2] + m.w * y[3];
          }
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) sN[(r0 + r) * kLd + c] = x[r];
      }
      __syncthreads();
      if (warp == 7 && g + 1 < p.group) scalars(g + 1);
      // ---- T = I - N diag b, T2 = -diag(b) N: four threads a row
      {
        const int r = tid & 63, c0 = (tid >> 6) * 16;
        const float br = sB[r];
        uint4* t = reinterpret_cast<uint4*>(a.b.T + item * 2 * 4096) + 8 * c0 + r;
        uint4* t2 = a.b.T2 ? reinterpret_cast<uint4*>(a.b.T2 + item * 2 * 4096) + 8 * c0 + r : nullptr;
#pragma unroll
        for (int j = 0; j < 16; j += 8) {
          float x[8], z[8];
#pragma unroll
          for (int d = 0; d < 8; d += 4) {
            const float4 m = *reinterpret_cast<const float4*>(sN + r * kLd + c0 + j + d);
            const float4 b = *reinterpret_cast<const float4*>(sB + c0 + j + d);
            const float mm[4] = {m.x, m.y, m.z, m.w}, bb[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const int col = c0 + j + d + k;
              x[d + k] = col < r ? -mm[k] * bb[k] : col == r ? 1.f : 0.f;
              z[d + k] = col < r ? -br * mm[k] : 0.f;
            }
          }
          store_split(t + 8 * j, x);
          if (t2) store_split(t2 + 8 * j, z);
        }
      }
    }
  }
  tc::tc_fence_before();
  __syncthreads();
  if (warp == 0) tc::tmem_dealloc(tmem, 64);
  if (kPart && a.part.beside && blockIdx.x + blockIdx.y + blockIdx.z == 0) wait_prerequisites();
}

bool map_rows(CUtensorMap* m, const void* base, int heads, int tokens) {
  const uint64_t dims[3] = {kW, (uint64_t)heads, (uint64_t)tokens}, str[2] = {kW * 2, (uint64_t)heads * kW * 2};
  const uint32_t box[3] = {64, 1, 64};
  return encode_bf16_map(m, base, 3, dims, str, box);
}
int launch_pairs(const Params& p, const ChunkBuffers& b, const Part& part, cudaStream_t st) {
  CUtensorMap tm_k, tm_q;
  if (!map_rows(&tm_k, p.k, p.key_heads, p.geo.total_tokens) || !map_rows(&tm_q, p.q, p.key_heads, p.geo.total_tokens))
    return PKDA_ERR_LAUNCH;
  PairParams a;
  a.p = p; a.b = b; a.part = part;
  const auto kernel = part.c1 ? gdr_pairs_kernel<true> : gdr_pairs_kernel<false>;
  if (!ensure_dynamic_smem(kernel, pairs::kSmem)) return PKDA_ERR_LAUNCH;
  begin_stage(kStageGdrPairs, st);
  const int rc = launch_kernel(kernel, part.c1 ? dim3(part.c1 - part.c0, p.key_heads, p.geo.n_seqs) : dim3(p.geo.total_chunks, p.key_heads), pairs::kThreads, pairs::kSmem, st, tm_k, tm_q, a);
  end_stage(st);
  return rc;
}

}  // namespace gdr
}  // namespace pkda
