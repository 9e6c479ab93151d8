// State scan and output of the chunked gated delta rule: one CTA per (sequence, value head), chunk after chunk.
//
// The state is held transposed, a value channel per thread and tensor-memory lane, so everything between two products stays
// in its lane: a thread reads its accumulator row, scales columns (tokens) by numbers, rounds and puts the result back into
// tensor memory as the A operand of the next product.  No operand that depends on the state passes through shared memory.
//   KS^T = S^T k^T            A: S^T in tensor memory, split        M 128 (v)  N 64 (token)    K 128 twice
//   E^T  = v^T T^T - (exp(G) KS)^T T^T       A: v by TMA, then -exp(G) KS^T in tensor memory; both split   K 64 five times
//   S'^T = exp(G_L) S^T + (exp(G_L - G) b E)^T k                    split      N 128 (k)       K 64 twice
//   o^T  = s exp(G) (S^T q^T) + (b E)^T P^T                 all but q split    N 64            K 128 twice, 64 three times
// (Every operand of o that was computed is split as well, so that its rounding to bf16 is all that it is off by: 1.7e-3 root mean
// square.  With S^T and P in one part each it was off by 2.1e-3 to 2.7e-3, for 4 % less time.)
// Three round trips (product, read, write back) are the chain of a chunk: KS, E, S.  2.8 us a chunk without saved states (128
// chunks of 16 heads: 353 us), 3.4 with them (434 us); that chain bounds a call of fewer units than SMs.  8 x 4,096 tokens of 16
// heads for a backward: 273 us for 1.61 GB, 0.90 of the copy rate.  The products that hang on none of them
// (v^T T^T, S^T q^T) are issued behind the one the threads wait for.
//
// Warps: 0..7 the state (fp32, 64 values a thread in registers; warp w has channels 32 (w % 4).. and half w / 4 of the keys or
// tokens), 8..11 the output (they read the accumulators that the others have left behind), 12 TMA, 13 the products,
// 14 the states that are saved.
// Tiles come two chunks deep.  Every wait is bounded: a warp that gives up sets the status word and leaves the loop, the
// others' waits then run out as well.
#include "gdr_tc.cuh"

namespace pkda {
namespace gdr {

namespace scan {
constexpr int kStages = 2;                      // tiles in flight
constexpr int oK = 0, oQ = 16384, oV = 32768;   // 2 blocks [64 tok][64 ch] each
constexpr int oT = 49152, oP = oT + 16384;      // [64][64] each: T hi, T lo, P hi, P lo
constexpr int oScal = oP + 16384;               // kScanScalars fp32
constexpr int kTx = oScal + kScanScalars * 4;
constexpr int kStage = oScal + 1024;
constexpr int oKeep = kStages * kStage;         // saving: a state on its way out, as it will lie
constexpr int kFront = 1024;                    // barriers, in front of the tiles, which lie on 1,024 bytes
constexpr int kSmem = kFront + oKeep, kSaveSmem = kSmem + 65536;  // (saving takes all the shared memory there is)
constexpr int kThreads = 512;   // (the last warp only makes up its warpgroup)
// Registers a thread: the state warps take what the others give up.  256 x 176 + 128 x 112 + 128 x 48 = the 512 x 128 of the launch.
constexpr int kStateRegs = 176, kOutRegs = 112, kRestRegs = 48;
constexpr int kStateWarps = 8, kOutWarps = 4;
// tensor memory columns
constexpr uint32_t cS = 0, cKS = 128, cQS = 192, cE = 256, cPU = 320, cSb = 384, kCols = 512;
// Operands take the columns of what is used up.  S^T: hi in cSb.., lo 64 further.  The corrections replace KS, the warps of each
// half of the tokens in their own 32 columns: 16 of hi, 16 of lo; b E follows them there.  The writes go where S^T's lo was.
constexpr uint32_t cW = cSb + 64;
__host__ __device__ constexpr uint32_t half_cols(int kk) { return 32 * (kk >> 1) + 8 * (kk & 1); }  // of a k-step of 16 tokens; lo 16 on
static_assert(kTx <= kStage && kStage % 1024 == 0 && kSaveSmem <= 232448, "shared memory of one SM");
// barriers, 8 bytes each
enum { bFull = 0, bEmpty = bFull + kStages, bSb = bEmpty + kStages, bKS, bR, bE, bW, bU, bS, bO, bOfree, bKeep, bKeepFree, bCount };
static_assert(8 * bCount + 4 <= kFront, "the address of the tensor memory lies behind the barriers");
}  // namespace scan

struct ScanParams {
  Params p;
  ChunkBuffers b;
  Part part;
  const float* S0;
  bf16* o;
  float* ST;
};

// 32 accumulator columns of this warp's lanes.
__device__ __forceinline__ void load32(uint32_t taddr, float (&v)[32]) {
  tc::tmem_ld32(taddr, v);
  tc::tmem_ld_wait();
}

template <bool kSave>
__global__ void __launch_bounds__(scan::kThreads, 1)
gdr_scan_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_q,
                const __grid_constant__ CUtensorMap tm_v, const ScanParams a) {
  wait_prerequisites();
  using namespace scan;
  extern __shared__ __align__(1024) unsigned char smem_scan[];
  const Params& p = a.p;
  const int H = p.geo.heads, n = blockIdx.x / H, h = blockIdx.x - n * H, hk = h / p.group;
  const SeqInfo sq = part_sequence(p.geo, a.part, n);
  const int tid = threadIdx.x, warp = (int)tc::uniform(tid >> 5), lane = tid & 31;
  const int q = warp & 3, hf = (warp >> 2) & 1, v = 32 * q + lane;  // this thread's value channel
  const uint32_t bars = smem_u32(smem_scan), base = bars + kFront, slot = bars + 8 * bCount;
  unsigned char* tiles = smem_scan + kFront;
  auto bar = [&](int b) { return bars + 8 * b; };
  if (warp == 0) tc::tmem_alloc(slot, kCols);
  if (tid == 32) {
    for (int s = 0; s < kStages; ++s) {
      tc::mbar_init(bar(bFull + s), 1);
      tc::mbar_init(bar(bEmpty + s), 1 + kStateWarps + kOutWarps);  // products, and who reads the scalars
    }
    for (int b : {(int)bSb, (int)bR, (int)bW, (int)bU}) tc::mbar_init(bar(b), kStateWarps);
    for (int b : {(int)bKS, (int)bE, (int)bS, (int)bO}) tc::mbar_init(bar(b), 1);
    tc::mbar_init(bar(bOfree), kOutWarps);
    tc::mbar_init(bar(bKeep), kStateWarps);
    tc::mbar_init(bar(bKeepFree), 1);
    tc::fence_barrier_init();
  }
  tc::tc_fence_before();
  __syncthreads();
  launch_dependents();
  tc::tc_fence_after();
  const uint32_t tmem = tc::uniform(*reinterpret_cast<volatile uint32_t*>(smem_scan + 8 * bCount));
  const uint32_t lanes = tmem + ((uint32_t)(32 * q) << 16);
  const size_t sbase = (size_t)blockIdx.x * kW * kW;
  bool ok = true;
  // Waits for phase `i` of a barrier (its i-th completion); all lanes of a warp together.
  auto wait = [&](int b, int i) { ok = __all_sync(0xffffffffu, ok && tc::mbar_wait(bar(b), i & 1)); };
  auto arrive = [&](int b) {  // one arrival a warp, after what its lanes did before
    __syncwarp();
    if (lane == 0) mbar_arrive(bar(b));
  };

  if (warp < kStateWarps) {
    tc::regs_up<kStateRegs>();
    // ------------------------------------------------------------------------------------------ the state
    float S[64];  // S[key 64 hf + j][v]
#pragma unroll
    for (int j = 0; j < 64; ++j) S[j] = a.S0 ? a.S0[sbase + (size_t)(64 * hf + j) * kW + v] : 0.f;
    for (int i = 0; i < sq.nchunks && ok; ++i) {
      const float* sc = reinterpret_cast<const float*>(tiles + (i % kStages) * kStage + oScal) + 32 * hf;
      uint32_t hi[32], lo[32];
#pragma unroll
      for (int j = 0; j < 32; ++j) split2(S[2 * j], S[2 * j + 1], hi[j], lo[j]);
      tc::tmem_st32(lanes + cSb + 32 * hf, hi);
      tc::tmem_st32(lanes + cSb + 64 + 32 * hf, lo);
      tc::tmem_st_wait();
      tc::tc_fence_before();
      arrive(bSb);
      if (kSave) {
        // The state leaves by one bulk copy, which a warp of its own issues: stores by the threads (64 KB at the rate of a store
        // path) held them up in front of their next wait.
        if (i > 0) wait(bKeepFree, i - 1);
        if (!ok) break;
        unsigned char* keep = tiles + oKeep + 8 * hf * kOctet * 2 + v * 16;
#pragma unroll
        for (int j = 0; j < 32; j += 4) {
          *reinterpret_cast<uint4*>(keep + j / 4 * kOctet * 2) = make_uint4(hi[j], hi[j + 1], hi[j + 2], hi[j + 3]);
          *reinterpret_cast<uint4*>(keep + kW * kW * 2 + j / 4 * kOctet * 2) = make_uint4(lo[j], lo[j + 1], lo[j + 2], lo[j + 3]);
        }
        tc::fence_proxy_async();
        arrive(bKeep);
      }
      wait(bFull + i % kStages, i / kStages);  // (the scalars; the products behind bKS have waited for the tiles too)
      wait(bKS, i);
      if (!ok) break;
      tc::tc_fence_after();
      {
        float x[32];
        uint32_t hi[16], lo[16];
        load32(lanes + cKS + 32 * hf, x);
#pragma unroll
        for (int j = 0; j < 32; j += 4) {
          const float4 g = *reinterpret_cast<const float4*>(sc + j);
          split2(-g.x * x[j], -g.y * x[j + 1], hi[j / 2], lo[j / 2]);
          split2(-g.z * x[j + 2], -g.w * x[j + 3], hi[j / 2 + 1], lo[j / 2 + 1]);
        }
        tc::tmem_st16(lanes + cKS + 32 * hf, hi);
        tc::tmem_st16(lanes + cKS + 32 * hf + 16, lo);
        tc::tmem_st_wait();
      }
      tc::tc_fence_before();
      arrive(bR);
      wait(bE, i);
      if (!ok) break;
      tc::tc_fence_after();
      {
        float x[32];
        uint32_t hi[16], lo[16];
        load32(lanes + cE + 32 * hf, x);
#pragma unroll
        for (int j = 0; j < 32; j += 4) {
          const float4 k = *reinterpret_cast<const float4*>(sc + 128 + j);
          split2(k.x * x[j], k.y * x[j + 1], hi[j / 2], lo[j / 2]);
          split2(k.z * x[j + 2], k.w * x[j + 3], hi[j / 2 + 1], lo[j / 2 + 1]);
        }
        tc::tmem_st16(lanes + cW + 32 * hf, hi);
        tc::tmem_st16(lanes + cW + 32 * hf + 16, lo);
        tc::tmem_st_wait();
        tc::tc_fence_before();
        arrive(bW);
        // b E for the output, while the state's product runs
#pragma unroll
        for (int j = 0; j < 32; j += 4) {
          const float4 b = *reinterpret_cast<const float4*>(sc + 64 + j);
          split2(b.x * x[j], b.y * x[j + 1], hi[j / 2], lo[j / 2]);
          split2(b.z * x[j + 2], b.w * x[j + 3], hi[j / 2 + 1], lo[j / 2 + 1]);
        }
        tc::tmem_st16(lanes + cKS + 32 * hf, hi);
        tc::tmem_st16(lanes + cKS + 32 * hf + 16, lo);
        tc::tmem_st_wait();
      }
      tc::tc_fence_before();
      arrive(bU);
      const float gl = reinterpret_cast<const float*>(tiles + (i % kStages) * kStage + oScal)[63];  // exp(G_L)
      arrive_behind_loads(bar(bEmpty + i % kStages), __float_as_uint(gl));
      wait(bS, i);
      if (!ok) break;
      tc::tc_fence_after();
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        float x[32];
        load32(lanes + cS + 64 * hf + 32 * half, x);
#pragma unroll
        for (int j = 0; j < 32; ++j) S[32 * half + j] = gl * S[32 * half + j] + x[j];
      }
      tc::tc_fence_before();
    }
    if (!ok) {
      if (lane == 0) atomicExch(a.b.status, 1);
    } else if (a.ST) {
#pragma unroll
      for (int j = 0; j < 64; ++j) a.ST[sbase + (size_t)(64 * hf + j) * kW + v] = S[j];
    }
  } else if (warp < kStateWarps + kOutWarps) {
    tc::regs_down<kOutRegs>();
    // ------------------------------------------------------------------------------------------ the output
    for (int i = 0; i < sq.nchunks && ok; ++i) {
      const float* sc = reinterpret_cast<const float*>(tiles + (i % kStages) * kStage + oScal);
      const int tok0 = sq.bos + i * kChunk, valid = min(kChunk, sq.len - i * kChunk);
      wait(bFull + i % kStages, i / kStages);
      wait(bO, i);
      if (!ok) break;
      tc::tc_fence_after();
      uint32_t out[32];
      const size_t item = (size_t)(sq.chunk0 + i) * H + h;
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        float x[32], y[32];
        tc::tmem_ld32(lanes + cQS + 32 * half, x);
        tc::tmem_ld32(lanes + cPU + 32 * half, y);
        tc::tmem_ld_wait();
#pragma unroll
        for (int j = 0; j < 32; j += 2) {
          const float2 g = *reinterpret_cast<const float2*>(sc + 32 * half + j);
          out[16 * half + j / 2] = pack_bf16(p.scale * g.x * x[j] + y[j], p.scale * g.y * x[j + 1] + y[j + 1]);
        }
        if (kSave) {
          load32(lanes + cE + 32 * half, x);
          bf16* keep = a.b.e + item * 2 * kW * 64 + 4 * half * kOctet + v * 8;
#pragma unroll
          for (int j = 0; j < 32; j += 8) {
            uint4 hi, lo;
            split2(x[j], x[j + 1], hi.x, lo.x);
            split2(x[j + 2], x[j + 3], hi.y, lo.y);
            split2(x[j + 4], x[j + 5], hi.z, lo.z);
            split2(x[j + 6], x[j + 7], hi.w, lo.w);
            *reinterpret_cast<uint4*>(keep + j / 8 * kOctet) = hi;
            *reinterpret_cast<uint4*>(keep + kW * 64 + j / 8 * kOctet) = lo;
          }
        }
      }
      tc::tc_fence_before();
      arrive(bOfree);
      {
        uint32_t seen = 0;
#pragma unroll
        for (int j = 0; j < 32; ++j) seen ^= out[j];
        arrive_behind_loads(bar(bEmpty + i % kStages), seen);
      }
      const size_t at = ((size_t)tok0 * H + h) * kW + v, step = (size_t)H * kW;
      unsigned short* po = reinterpret_cast<unsigned short*>(a.o) + at;
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
    // ------------------------------------------------------------------------------------------ TMA
    if (lane == 0) {
      int i = 0;
      for (; i < sq.nchunks; ++i) {
        const int s = i % kStages, tok0 = sq.bos + i * kChunk;
        if (i >= kStages) {
          ok = tc::mbar_wait(bar(bEmpty + s), (i / kStages - 1) & 1);
          if (!ok) break;
        }
        const uint32_t st = base + s * kStage, full = bar(bFull + s);
        const size_t item = (size_t)(sq.chunk0 + i) * H + h;
        tc::mbar_expect_tx(full, kTx);
#pragma unroll
        for (int b = 0; b < 2; ++b) tc::tma_load_3d(st + oK + 8192 * b, &tm_k, full, 64 * b, hk, tok0);
        tc::bulk_load(st + oT, a.b.T + item * 2 * 4096, 16384, full);
#pragma unroll
        for (int b = 0; b < 2; ++b) tc::tma_load_3d(st + oV + 8192 * b, &tm_v, full, 64 * b, h, tok0);
        tc::bulk_load(st + oScal, a.b.scal + item * kScalars, kScanScalars * 4, full);
#pragma unroll
        for (int b = 0; b < 2; ++b) tc::tma_load_3d(st + oQ + 8192 * b, &tm_q, full, 64 * b, hk, tok0);
        tc::bulk_load(st + oP, a.b.P + item * 2 * 4096, 16384, full);
      }
      if (!ok) {
        atomicExch(a.b.status, 1);
        // copies in flight have to land before the CTA's shared memory goes to another
        for (int j = i > kStages ? i - kStages : 0; j < i; ++j) tc::mbar_wait(bar(bFull + j % kStages), (j / kStages) & 1);
      }
    }
  } else if (warp == kStateWarps + kOutWarps + 1) {
    // ------------------------------------------------------------------------------------------ the products
    constexpr uint32_t kk128 = tc::idesc_bf16(128, 64, false, false), vt = tc::idesc_bf16(128, 64, true, false),
                       wk = tc::idesc_bf16(128, 128, false, true);
    for (int i = 0; i < sq.nchunks && ok; ++i) {
      const uint32_t st = tc::uniform(base + (i % kStages) * kStage);  // (descriptors in uniform registers: pkda_tc.cuh)
      const int valid = min(kChunk, sq.len - i * kChunk);
      wait(bFull + i % kStages, i / kStages);
      if (!ok) break;
      if (valid < kChunk) {
        unsigned char* t = tiles + (i % kStages) * kStage;
        zero_rows(t + oK, 8192, valid);
        zero_rows(t + oQ, 8192, valid);
        zero_rows(t + oV, 8192, valid);
        tc::fence_proxy_async();
        __syncwarp();
      }
      if (i > 0) wait(bO, i - 1);  // (P u of the chunk before reads its u where k S goes)
      wait(bSb, i);
      if (!ok) break;
      tc::tc_fence_after();
      if (tc::elect_one()) {
#pragma unroll
        for (int kk = 0; kk < 16; ++kk)
          tc::umma_bf16_ta(tmem + cKS, tmem + cSb + 8 * kk, tc::desc_kmajor(st + oK + ((kk >> 2) & 1) * 8192 + (kk & 3) * 32), kk128, kk > 0);
        tc::umma_commit(bar(bKS));
      }
      __syncwarp();
      if (i > 0) wait(bOfree, i - 1);  // the output warps have read what the chunk before left
      if (!ok) break;
      tc::tc_fence_after();
      if (tc::elect_one()) {
#pragma unroll
        for (int kk = 0; kk < 8; ++kk)
          tc::umma_bf16(tmem + cE, tc::desc_mnmajor(st + oV + (kk & 3) * 2048, 8192),
                        pair_desc(st + oT + (kk >> 2) * 8192, kk & 3), vt, kk > 0);
#pragma unroll
        for (int kk = 0; kk < 16; ++kk)
          tc::umma_bf16_ta(tmem + cQS, tmem + cSb + 8 * kk, tc::desc_kmajor(st + oQ + ((kk >> 2) & 1) * 8192 + (kk & 3) * 32), kk128, kk > 0);
      }
      __syncwarp();
      wait(bR, i);
      if (!ok) break;
      tc::tc_fence_after();
      if (tc::elect_one()) {
#pragma unroll
        for (int kk = 0; kk < 12; ++kk)  // hi T hi, hi T lo, lo T hi
          tc::umma_bf16_ta(tmem + cE, tmem + cKS + half_cols(kk & 3) + (kk < 8 ? 0 : 16),
                           pair_desc(st + oT + (kk >> 2 == 1 ? 8192 : 0), kk & 3), kk128, 1);
        tc::umma_commit(bar(bE));
      }
      __syncwarp();
      wait(bW, i);
      if (!ok) break;
      tc::tc_fence_after();
      if (tc::elect_one()) {
#pragma unroll
        for (int kk = 0; kk < 8; ++kk)
          tc::umma_bf16_ta(tmem + cS, tmem + cW + half_cols(kk & 3) + (kk < 4 ? 0 : 16),
                           tc::desc_mnmajor(st + oK + (kk & 3) * 2048, 8192), wk, kk > 0);
        tc::umma_commit(bar(bS));
      }
      __syncwarp();
      wait(bU, i);
      if (!ok) break;
      tc::tc_fence_after();
      if (tc::elect_one()) {
#pragma unroll
        for (int kk = 0; kk < 12; ++kk)  // hi P hi, hi P lo, lo P hi
          tc::umma_bf16_ta(tmem + cPU, tmem + cKS + half_cols(kk & 3) + (kk < 8 ? 0 : 16),
                           pair_desc(st + oP + (kk >> 2 == 1 ? 8192 : 0), kk & 3), kk128, kk > 0);
        tc::umma_commit(bar(bO));
        tc::umma_commit(bar(bEmpty + i % kStages));
      }
      __syncwarp();
    }
    if (!ok && lane == 0) atomicExch(a.b.status, 1);
  } else if (kSave && warp == kStateWarps + kOutWarps + 2) {
    // ------------------------------------------------------------------------------------------ saved states out
    for (int i = 0; i < sq.nchunks && ok; ++i) {
      wait(bKeep, i);
      if (ok && lane == 0) {
        tc::bulk_store(a.b.h + ((size_t)(sq.chunk0 + i) * H + h) * 2 * kW * kW, base + oKeep, 65536);
        tc::bulk_commit();
        tc::bulk_wait_read();
        mbar_arrive(bar(bKeepFree));
      }
      __syncwarp();
    }
    tc::bulk_wait_all();  // (it must have left before the CTA's shared memory goes to another)
    if (!ok && lane == 0) atomicExch(a.b.status, 1);
  }
  }
  tc::tc_fence_before();
  __syncthreads();
  if (warp == 0) tc::tmem_dealloc(tmem, kCols);
  // If any kernel of the call gave up (this CTA included), the first output row of this unit and its state become NaN, so that a
  // caller who never reads the status word cannot take a partial result for a complete one.
  if (warp == 1 && *reinterpret_cast<volatile int*>(a.b.status) != 0) {
    if (sq.len > 0) mark_failed(a.o + ((size_t)sq.bos * H + h) * kW, kW);
    if (a.ST) mark_failed(a.ST + sbase, kW * kW);
  }
}

int launch_scan(const Params& p, const ChunkBuffers& b, const Part& part, const float* S0, bf16* o, float* ST, cudaStream_t st) {
  CUtensorMap tm_k, tm_q, tm_v;
  const int tok = p.geo.total_tokens;
  if (!map_rows(&tm_k, p.k, p.key_heads, tok) || !map_rows(&tm_q, p.q, p.key_heads, tok) ||
      !map_rows(&tm_v, p.v, p.geo.heads, tok))
    return PKDA_ERR_LAUNCH;
  ScanParams a;
  a.p = p; a.b = b; a.part = part; a.S0 = S0; a.o = o; a.ST = ST;
  const auto kernel = b.h ? gdr_scan_kernel<true> : gdr_scan_kernel<false>;
  const int smem = b.h ? scan::kSaveSmem : scan::kSmem;
  if (!ensure_dynamic_smem(kernel, smem)) return PKDA_ERR_LAUNCH;
  begin_stage(kStageGdrScan, st);
  const int rc = launch_kernel(!part.ordinary, kernel, p.geo.n_seqs * p.geo.heads, scan::kThreads, smem, st, tm_k, tm_q, tm_v, a);
  end_stage(st);
  return rc;
}

}  // namespace gdr
}  // namespace pkda
