// Reverse state scan of the chunked gated delta rule: one CTA per (sequence, value head), last chunk first.
//
// The mirror of the forward scan (gdr_scan_tc.cu), with the state's cotangent transposed in the lanes of tensor memory:
//   KD^T = dS'^T k^T           du^T = exp(G_L - G) KD^T + do^T P
//   y^T  = du^T - (du^T)(diag(b) N)                        (T2 holds -diag(b) N; the du beside it stays in fp32)
//   dS^T = exp(G_L) dS'^T + do^T (s exp(G) q) - (exp(G) b y)^T k
// Three round trips again: KD, y, dS.  do^T P and do^T (s exp(G) q) hang on none of them and are issued in their shadow.  dS' of
// every chunk and y are left for the gradients (gdr_grad_tc.cu), split like every computed operand here; dv = b y leaves.
// 8 x 4,096 tokens of 16 heads (64 chunks): 281 us for 1.61 GB, 0.87 of the copy rate; stores by the threads instead of bulk
// copies 324.  16 units alone take 4.1 us a chunk.
//
// Warps: 0..7 the cotangent, 8..11 scale q (hi in place) and carry y and dv out, 12 TMA, 13 the products, 14 the cotangents out.
#include "gdr_tc.cuh"

namespace pkda {
namespace gdr {

namespace rscan {
constexpr int kStages = 2;
constexpr int oK = 0, oDo = 16384, oQ = 32768, oT2 = 49152, oP = 65536, oScal = 81920;
constexpr int kTx = oScal + kScanScalars * 4;
constexpr int kStage = oScal + 1024;
constexpr int oQlo = kStages * kStage;          // lo of the scaled q of a chunk
constexpr int oKeep = oQlo + 16384;             // half of a cotangent (hi, then lo) on its way out, as it will lie
constexpr int oBar = oKeep + 32768;
constexpr int kSmem = oBar + 256 + 1024;
constexpr int kThreads = 512;
constexpr int kStateWarps = 8, kOutWarps = 4;
constexpr int kStateRegs = 184, kOutRegs = 96, kRestRegs = 48;  // 256 x 184 + 128 x 96 + 128 x 48 = the 512 x 128 of the launch
constexpr uint32_t cS = 0, cKD = 128, cY0 = 192, cY = 256, cDb = 320, cW = cDb + 64, kCols = 512;
__host__ __device__ constexpr uint32_t half_cols(int kk) { return 32 * (kk >> 1) + 8 * (kk & 1); }  // of a k-step of 16 tokens; lo 16 on
static_assert(kStage % 1024 == 0 && kSmem <= 232448, "shared memory of one SM");
enum { bFull = 0, bEmpty = bFull + kStages, bQ = bEmpty + kStages, bDb = bQ + kStages, bKD, bDU, bY, bW, bS, bYout, bOfree, bKeep, bKeepFree, bCount };
}  // namespace rscan

struct ReverseParams {
  Params p;
  ChunkBuffers b;
  GradBuffers g;
  bf16* dv;
  const float* dST;
  float* dS0;
  Part part;
};

__global__ void __launch_bounds__(rscan::kThreads, 1)
gdr_scan_bwd_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_q,
                    const __grid_constant__ CUtensorMap tm_do, const ReverseParams a) {
  wait_prerequisites();
  using namespace rscan;
  extern __shared__ unsigned char smem_raw[];
  const Params& p = a.p;
  const int H = p.geo.heads, n = blockIdx.x / H, h = blockIdx.x - n * H, hk = h / p.group;
  const SeqInfo sq = part_sequence(p.geo, a.part, n);
  const int tid = threadIdx.x, warp = (int)tc::uniform(tid >> 5), lane = tid & 31;
  const int q = warp & 3, hf = (warp >> 2) & 1, v = 32 * q + lane;
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  unsigned char* tiles = smem_raw + (base - smem_u32(smem_raw));
  const uint32_t bars = base + oBar, slot = bars + 8 * bCount;
  auto bar = [&](int b) { return bars + 8 * b; };
  if (warp == 0) tc::tmem_alloc(slot, kCols);
  if (tid == 32) {
    for (int s = 0; s < kStages; ++s) {
      tc::mbar_init(bar(bFull + s), 1);
      tc::mbar_init(bar(bEmpty + s), 1 + kStateWarps + kOutWarps);
      tc::mbar_init(bar(bQ + s), kOutWarps);
    }
    for (int b : {(int)bDb, (int)bDU, (int)bW, (int)bYout}) tc::mbar_init(bar(b), kStateWarps);
    for (int b : {(int)bKD, (int)bY, (int)bS}) tc::mbar_init(bar(b), 1);
    tc::mbar_init(bar(bOfree), kOutWarps);
    tc::mbar_init(bar(bKeep), kStateWarps);
    tc::mbar_init(bar(bKeepFree), 1);
    tc::fence_barrier_init();
  }
  tc::tc_fence_before();
  __syncthreads();
  launch_dependents();
  tc::tc_fence_after();
  const uint32_t tmem = tc::uniform(*reinterpret_cast<volatile uint32_t*>(tiles + oBar + 8 * bCount));
  const uint32_t lanes = tmem + ((uint32_t)(32 * q) << 16);
  const size_t sbase = (size_t)blockIdx.x * kW * kW;
  const int last = sq.nchunks - 1;  // step j works on chunk last - j
  bool ok = true;
  auto wait = [&](int b, int i) { ok = __all_sync(0xffffffffu, ok && tc::mbar_wait(bar(b), i & 1)); };
  auto arrive = [&](int b) {
    __syncwarp();
    if (lane == 0) mbar_arrive(bar(b));
  };

  if (warp < kStateWarps) {
    tc::regs_up<kStateRegs>();
    // -------------------------------------------------------------------------------------- the state's cotangent
    float S[64];  // dS[key 64 hf + j][v]
#pragma unroll
    for (int j = 0; j < 64; ++j) S[j] = a.dST ? a.dST[sbase + (size_t)(64 * hf + j) * kW + v] : 0.f;
    auto keep_half = [&](const uint32_t (&w)[32]) {
      unsigned char* keep = tiles + oKeep + 8 * hf * kOctet * 2 + v * 16;
#pragma unroll
      for (int j = 0; j < 32; j += 4)
        *reinterpret_cast<uint4*>(keep + j / 4 * kOctet * 2) = make_uint4(w[j], w[j + 1], w[j + 2], w[j + 3]);
      tc::fence_proxy_async();
      arrive(bKeep);
    };
    for (int i = 0; i < sq.nchunks && ok; ++i) {
      const int s = i % kStages;
      const float* sc = reinterpret_cast<const float*>(tiles + s * kStage + oScal) + 32 * hf;
      {
        uint32_t hi[32], lo[32];
#pragma unroll
        for (int j = 0; j < 32; ++j) split2(S[2 * j], S[2 * j + 1], hi[j], lo[j]);
        tc::tmem_st32(lanes + cDb + 32 * hf, hi);
        tc::tmem_st32(lanes + cDb + 64 + 32 * hf, lo);
        tc::tmem_st_wait();
        tc::tc_fence_before();
        arrive(bDb);
        // hi leaves now, lo while y is on its way (gdr_scan_tc.cu); there is room for one of them
        if (i > 0) wait(bKeepFree, 2 * i - 1);
        if (!ok) break;
        keep_half(hi);
      }
      wait(bFull + s, i / kStages);
      wait(bKD, i);
      if (!ok) break;
      tc::tc_fence_after();
      float du[32];
      {
        float x[32];
        uint32_t hi[16], lo[16];
        tc::tmem_ld32(lanes + cKD + 32 * hf, x);
        tc::tmem_ld32(lanes + cY0 + 32 * hf, du);
        tc::tmem_ld_wait();
#pragma unroll
        for (int j = 0; j < 32; j += 4) {
          const float4 k = *reinterpret_cast<const float4*>(sc + 192 + j);
          du[j] += k.x * x[j];
          du[j + 1] += k.y * x[j + 1];
          du[j + 2] += k.z * x[j + 2];
          du[j + 3] += k.w * x[j + 3];
          split2(du[j], du[j + 1], hi[j / 2], lo[j / 2]);
          split2(du[j + 2], du[j + 3], hi[j / 2 + 1], lo[j / 2 + 1]);
        }
        tc::tmem_st16(lanes + cKD + 32 * hf, hi);
        tc::tmem_st16(lanes + cKD + 32 * hf + 16, lo);
        tc::tmem_st_wait();
      }
      tc::tc_fence_before();
      arrive(bDU);
      {
        uint32_t hi[32], lo[32];
#pragma unroll
        for (int j = 0; j < 32; ++j) split2(S[2 * j], S[2 * j + 1], hi[j], lo[j]);
        wait(bKeepFree, 2 * i);
        if (!ok) break;
        keep_half(lo);
      }
      wait(bY, i);
      if (!ok) break;
      tc::tc_fence_after();
      {
        float x[32];
        uint32_t hi[16], lo[16];
        tc::tmem_ld32(lanes + cY + 32 * hf, x);
        tc::tmem_ld_wait();
#pragma unroll
        for (int j = 0; j < 32; j += 4) {
          const float4 g = *reinterpret_cast<const float4*>(sc + j), b = *reinterpret_cast<const float4*>(sc + 64 + j);
          x[j] += du[j];
          x[j + 1] += du[j + 1];
          x[j + 2] += du[j + 2];
          x[j + 3] += du[j + 3];
          split2(-g.x * b.x * x[j], -g.y * b.y * x[j + 1], hi[j / 2], lo[j / 2]);
          split2(-g.z * b.z * x[j + 2], -g.w * b.w * x[j + 3], hi[j / 2 + 1], lo[j / 2 + 1]);
        }
        tc::tmem_st16(lanes + cW + 32 * hf, hi);
        tc::tmem_st16(lanes + cW + 32 * hf + 16, lo);
        tc::tmem_st_wait();
        tc::tc_fence_before();
        arrive(bW);
        tc::tmem_st32(lanes + cY + 32 * hf, x);  // y, for the warps that carry it out
        tc::tmem_st_wait();
        tc::tc_fence_before();
        arrive(bYout);
      }
      const float gl = reinterpret_cast<const float*>(tiles + s * kStage + oScal)[63];
      arrive_behind_loads(bar(bEmpty + s), __float_as_uint(gl));
      wait(bS, i);
      if (!ok) break;
      tc::tc_fence_after();
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        float x[32];
        tc::tmem_ld32(lanes + cS + 64 * hf + 32 * half, x);
        tc::tmem_ld_wait();
#pragma unroll
        for (int j = 0; j < 32; ++j) S[32 * half + j] = gl * S[32 * half + j] + x[j];
      }
      tc::tc_fence_before();
    }
    if (!ok) {
      if (lane == 0) atomicExch(a.b.status, 1);
    } else if (a.dS0) {
#pragma unroll
      for (int j = 0; j < 64; ++j) a.dS0[sbase + (size_t)(64 * hf + j) * kW + v] = S[j];
    }
  } else if (warp < kStateWarps + kOutWarps) {
    tc::regs_down<kOutRegs>();
    // ------------------------------------------------------------------------------------------ s exp(G) q, y, dv
    for (int i = 0; i < sq.nchunks && ok; ++i) {
      const int s = i % kStages, c = last - i, tok0 = sq.bos + c * kChunk, valid = min(kChunk, sq.len - c * kChunk);
      unsigned char* st = tiles + s * kStage;
      const float* sc = reinterpret_cast<const float*>(st + oScal);
      wait(bFull + s, i / kStages);
      if (i > 0) wait(bS, i - 1);  // (the products of the chunk before have read the lo part)
      if (!ok) break;
#pragma unroll 2
      for (int x = tid - 32 * kStateWarps; x < kChunk * 16; x += 32 * kOutWarps) {  // 16-byte pieces: 8 channels of a token
        const int r = x >> 4, pc = x & 15;
        uint4* at = reinterpret_cast<uint4*>(st + oQ + (pc >> 3) * 8192 + r * 128 + ((pc & 7) << 4));
        const uint4 in = *at;
        const float f = p.scale * sc[r];
        uint4 hi = make_uint4(0, 0, 0, 0), lo = hi;
        if (r < valid) {
          const float2 e0 = unpack_bf16(in.x), e1 = unpack_bf16(in.y), e2 = unpack_bf16(in.z), e3 = unpack_bf16(in.w);
          split2(f * e0.x, f * e0.y, hi.x, lo.x);
          split2(f * e1.x, f * e1.y, hi.y, lo.y);
          split2(f * e2.x, f * e2.y, hi.z, lo.z);
          split2(f * e3.x, f * e3.y, hi.w, lo.w);
        }
        *at = hi;
        *reinterpret_cast<uint4*>(tiles + oQlo + (pc >> 3) * 8192 + r * 128 + ((pc & 7) << 4)) = lo;
      }
      tc::fence_proxy_async();
      arrive(bQ + s);
      wait(bYout, i);
      if (!ok) break;
      tc::tc_fence_after();
      uint32_t out[32];
      bf16* keep = a.g.y + ((size_t)(sq.chunk0 + c) * H + h) * 2 * kW * 64 + v * 8;
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        float x[32];
        tc::tmem_ld32(lanes + cY + 32 * half, x);
        tc::tmem_ld_wait();
#pragma unroll
        for (int j = 0; j < 32; j += 8) {
          uint4 hi, lo;
          split2(x[j], x[j + 1], hi.x, lo.x);
          split2(x[j + 2], x[j + 3], hi.y, lo.y);
          split2(x[j + 4], x[j + 5], hi.z, lo.z);
          split2(x[j + 6], x[j + 7], hi.w, lo.w);
          *reinterpret_cast<uint4*>(keep + (4 * half + j / 8) * kOctet) = hi;
          *reinterpret_cast<uint4*>(keep + kW * 64 + (4 * half + j / 8) * kOctet) = lo;
        }
#pragma unroll
        for (int j = 0; j < 32; j += 2) {
          const float2 b = *reinterpret_cast<const float2*>(sc + 64 + 32 * half + j);
          out[16 * half + j / 2] = pack_bf16(b.x * x[j], b.y * x[j + 1]);
        }
      }
      tc::tc_fence_before();
      arrive(bOfree);
      {
        uint32_t seen = 0;
#pragma unroll
        for (int j = 0; j < 32; ++j) seen ^= out[j];
        arrive_behind_loads(bar(bEmpty + s), seen);
      }
      unsigned short* po = reinterpret_cast<unsigned short*>(a.dv) + ((size_t)tok0 * H + h) * kW + v;
      const size_t step = (size_t)H * kW;
      if (valid == kChunk) {
#pragma unroll
        for (int j = 0; j < kChunk; ++j) {
          *po = (unsigned short)(out[j / 2] >> (16 * (j & 1)));
          po += step;
        }
      } else {
#pragma unroll
        for (int j = 0; j < kChunk; ++j)
          if (j < valid) po[j * step] = (unsigned short)(out[j / 2] >> (16 * (j & 1)));
      }
    }
    if (!ok && lane == 0) atomicExch(a.b.status, 1);
  } else {
    tc::regs_down<kRestRegs>();
    if (warp == kStateWarps + kOutWarps) {
      // ---------------------------------------------------------------------------------------- TMA
      if (lane == 0) {
        int i = 0;
        for (; i < sq.nchunks; ++i) {
          const int s = i % kStages, c = last - i, tok0 = sq.bos + c * kChunk;
          if (i >= kStages) {
            ok = tc::mbar_wait(bar(bEmpty + s), (i / kStages - 1) & 1);
            if (!ok) break;
          }
          const uint32_t st = base + s * kStage, full = bar(bFull + s);
          const size_t item = (size_t)(sq.chunk0 + c) * H + h;
          tc::mbar_expect_tx(full, kTx);
#pragma unroll
          for (int b = 0; b < 2; ++b) {
            tc::tma_load_3d(st + oK + 8192 * b, &tm_k, full, 64 * b, hk, tok0);
            tc::tma_load_3d(st + oDo + 8192 * b, &tm_do, full, 64 * b, h, tok0);
            tc::tma_load_3d(st + oQ + 8192 * b, &tm_q, full, 64 * b, hk, tok0);
          }
          tc::bulk_load(st + oP, a.b.P + item * 2 * 4096, 16384, full);
          tc::bulk_load(st + oT2, a.b.T2 + item * 2 * 4096, 16384, full);
          tc::bulk_load(st + oScal, a.b.scal + item * kScalars, kScanScalars * 4, full);
        }
        if (!ok) {
          atomicExch(a.b.status, 1);
          for (int j = i > kStages ? i - kStages : 0; j < i; ++j) tc::mbar_wait(bar(bFull + j % kStages), (j / kStages) & 1);
        }
      }
    } else if (warp == kStateWarps + kOutWarps + 1) {
      // ---------------------------------------------------------------------------------------- the products
      constexpr uint32_t kd = tc::idesc_bf16(128, 64, false, false), dop = tc::idesc_bf16(128, 64, true, true),
                         dut = tc::idesc_bf16(128, 64, false, true), doq = tc::idesc_bf16(128, 128, true, true),
                         wk = tc::idesc_bf16(128, 128, false, true);
      for (int i = 0; i < sq.nchunks && ok; ++i) {
        const int s = i % kStages, valid = min(kChunk, sq.len - (last - i) * kChunk);
        const uint32_t b0 = tc::uniform(base), st = b0 + s * kStage;
        wait(bFull + s, i / kStages);
        if (!ok) break;
        if (valid < kChunk) {
          zero_rows(tiles + s * kStage + oK, 8192, valid);
          zero_rows(tiles + s * kStage + oDo, 8192, valid);
          tc::fence_proxy_async();
          __syncwarp();
        }
        if (tc::elect_one()) {
#pragma unroll
          for (int kk = 0; kk < 8; ++kk)
            tc::umma_bf16(tmem + cY0, tc::desc_mnmajor(st + oDo + (kk & 3) * 2048, 8192),
                          pair_desc_t(st + oP + (kk >> 2) * 8192, kk & 3), dop, kk > 0);
        }
        __syncwarp();
        wait(bDb, i);
        if (!ok) break;
        tc::tc_fence_after();
        if (tc::elect_one()) {
#pragma unroll
          for (int kk = 0; kk < 16; ++kk)
            tc::umma_bf16_ta(tmem + cKD, tmem + cDb + 8 * kk, tc::desc_kmajor(st + oK + ((kk >> 2) & 1) * 8192 + (kk & 3) * 32), kd, kk > 0);
          tc::umma_commit(bar(bKD));
        }
        __syncwarp();
        wait(bQ + s, i / kStages);
        if (!ok) break;
        if (tc::elect_one()) {
#pragma unroll
          for (int kk = 0; kk < 8; ++kk)
            tc::umma_bf16(tmem + cS, tc::desc_mnmajor(st + oDo + (kk & 3) * 2048, 8192),
                          tc::desc_mnmajor((kk < 4 ? st + oQ : b0 + oQlo) + (kk & 3) * 2048, 8192), doq, kk > 0);
        }
        __syncwarp();
        if (i > 0) wait(bOfree, i - 1);
        wait(bDU, i);
        if (!ok) break;
        tc::tc_fence_after();
        if (tc::elect_one()) {
#pragma unroll
          for (int kk = 0; kk < 12; ++kk)
            tc::umma_bf16_ta(tmem + cY, tmem + cKD + half_cols(kk & 3) + (kk < 8 ? 0 : 16),
                             pair_desc_t(st + oT2 + (kk >> 2 == 1 ? 8192 : 0), kk & 3), dut, kk > 0);
          tc::umma_commit(bar(bY));
        }
        __syncwarp();
        wait(bW, i);
        if (!ok) break;
        tc::tc_fence_after();
        if (tc::elect_one()) {
#pragma unroll
          for (int kk = 0; kk < 8; ++kk)
            tc::umma_bf16_ta(tmem + cS, tmem + cW + half_cols(kk & 3) + (kk < 4 ? 0 : 16),
                             tc::desc_mnmajor(st + oK + (kk & 3) * 2048, 8192), wk, 1);
          tc::umma_commit(bar(bS));
          tc::umma_commit(bar(bEmpty + s));
        }
        __syncwarp();
      }
      if (!ok && lane == 0) atomicExch(a.b.status, 1);
    } else if (warp == kStateWarps + kOutWarps + 2) {
      // ---------------------------------------------------------------------------------------- cotangents out
      for (int i = 0; i < 2 * sq.nchunks && ok; ++i) {
        wait(bKeep, i);
        if (ok && lane == 0) {
          tc::bulk_store(a.g.dh + (((size_t)(sq.chunk0 + last - i / 2) * H + h) * 2 + (i & 1)) * kW * kW, base + oKeep, 32768);
          tc::bulk_commit();
          tc::bulk_wait_read();
          mbar_arrive(bar(bKeepFree));
        }
        __syncwarp();
      }
      tc::bulk_wait_all();  // (they must have left before the CTA's shared memory goes to another)
      if (!ok && lane == 0) atomicExch(a.b.status, 1);
    }
  }
  tc::tc_fence_before();
  __syncthreads();
  if (warp == 0) tc::tmem_dealloc(tmem, kCols);
  if (warp == 1 && *reinterpret_cast<volatile int*>(a.b.status) != 0) {  // (as in the forward scan)
    if (sq.len > 0) mark_failed(a.dv + ((size_t)sq.bos * H + h) * kW, kW);
    if (a.dS0) mark_failed(a.dS0 + sbase, kW * kW);
  }
}

int launch_scan_bwd(const Params& p, const ChunkBuffers& b, const GradBuffers& g, const Part& part, const bf16* d_o, const float* dST, bf16* dv,
                    float* dS0, cudaStream_t st) {
  const int tok = p.geo.total_tokens;
  CUtensorMap tm_k, tm_q, tm_do;
  if (!map_rows(&tm_k, p.k, p.key_heads, tok) || !map_rows(&tm_q, p.q, p.key_heads, tok) ||
      !map_rows(&tm_do, d_o, p.geo.heads, tok))
    return PKDA_ERR_LAUNCH;
  ReverseParams a;
  a.p = p; a.b = b; a.g = g; a.part = part; a.dv = dv; a.dST = dST; a.dS0 = dS0;
  if (!ensure_dynamic_smem(gdr_scan_bwd_kernel, rscan::kSmem)) return PKDA_ERR_LAUNCH;
  begin_stage(kStageGdrScanBwd, st);
  const int rc = launch_kernel(!part.ordinary, gdr_scan_bwd_kernel, p.geo.n_seqs * p.geo.heads, rscan::kThreads, rscan::kSmem, st, tm_k, tm_q, tm_do, a);
  end_stage(st);
  return rc;
}

}  // namespace gdr
}  // namespace pkda
