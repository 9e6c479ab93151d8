// Linear attention on tcgen05: one CTA walks over the chunks of a (sequence, head), or of a segment of it, forwards or backwards.
//
// With a chunk's reads x, keys y, values z (la_common.cuh), R the state in front of it, r_a = read 2^(decay of the chunk up to read a) and
// D_ab = r_a / read f_b (f_b = 2^-(the decay up to b), the pairs' decay with the chunk's start as reference):
//   P    = c / read (x y^T) f                 M 64 (reads)   N 64     K D            both as they are
//   QS^T = R^T x^T                            M 128 (z)      N 64     K D twice      R^T in two parts, in tensor memory
//   PV^T = z^T P^T                            M 128 (z)      N 64     K 64 twice     P in two parts, through shared memory
//   KV^T = z^T (w y)                          M 128 (z)      N D      K 64 twice     w y in two parts, through shared memory
//   out  = r (QS + PV),   R' = decay R + KV
// QS and PV share an accumulator, and two take turns, except where the reads of the state alone are wanted too (for the gate's gradient):
// then two of QS take turns.
// The state is held transposed, a channel of z per thread and tensor-memory lane, in fp32 registers; only the sum R' waits for the
// chunk before, so the products of a chunk run while the threads work on their neighbours'.
//
// Precision.  x, y, z are bf16 and enter as they are.  What is computed (P, R, w y) is split in two bf16 parts, off by 2^-17 of it at
// most, so that bf16 results are off by their own rounding and fp32 ones (states, the gate's gradient) by a few 2^-19.  A chunk's decay
// multiplies the state in two parts too: rounded once, a head of one decay would gain the same 2^-25 in every chunk.
//
// Warps: 0..7 the state (warp w has lanes 32 (w % 4).. and half w / 4 of the keys), 8..11 the output, 12..19 the weighted keys and the
// pairs, 20 tiles by TMA and a chunk's scalars, 21 and 22 the products (two warps, so that neither stands in front of what the other could
// issue), 23 u and the results' way out.  Every wait is bounded: a warp that gives up sets the status word and leaves its loop, the
// others' waits then run out as well.
//
// Bound by the instructions of its roles: 2.2 to 2.4 us a chunk with the SMs all at work, 2.8 with the gate's gradient, where the products
// take 0.9 and the bytes 1.5 at the copy rate (8 x 4,096 tokens of 16 heads: forward 151 us on 128 SMs, 3.6 TB/s; backward 521).
#include "la_tc.cuh"

#include <type_traits>

namespace pkda {
namespace la {

using gdr::arrive_behind_loads;
using gdr::mark_failed;
using gdr::mbar_arrive;

namespace {

template <int D> struct Cfg {
  static constexpr int kTile = kChunk * D * 2;
  static constexpr int kStages = D == 128 ? 3 : 5;
  static constexpr int oX = 0, oY = kTile, oZ = 2 * kTile, kStage = 3 * kTile;
  // Behind the stages: two slots that take u of a chunk and then its results, the lo parts of the weighted keys (their hi parts take the
  // keys' place), P hi and lo, and the scalars of twice as many chunks (who reads them last is two chunks behind the tiles' readers).
  static constexpr int oU = kStages * kStage, oYlo = oU + 2 * kTile, oP = oYlo + kTile, oScal = oP + 16384;
  static constexpr int kRing = 2 * kStages, kScal = 384 * 4;
  static constexpr int kFront = 1024;  // barriers, in front of the tiles, which lie on 1,024 bytes
  static constexpr int kSmem = kFront + oScal + kRing * kScal;
  // tensor memory columns
  static constexpr uint32_t cKV = 0, cR = D, cQK = 2 * D, cW = cQK + 64, cO = cQK + 128, kCols = 512;
  static_assert(kSmem <= 232448 && cO + 128 <= kCols, "shared and tensor memory of one SM");
  enum { bFull = 0, bEmpty = bFull + kStages, bScal = bEmpty + kStages, bU = bScal + kRing, bOut = bU + 2, bKV = bOut + 2, bO = bKV + 2, bP = bO + 2, bYw = bP + 2,
         bQK = bYw + 2, bQKfree = bQK + 2, bOfree = bQKfree + 2, bKVfree = bOfree + 2, bQS, bR, bCount };
  static_assert(8 * bCount + 4 <= kFront, "the address of the tensor memory lies behind the barriers");
};
constexpr int kThreads = 768;
constexpr int kStateWarps = 8, kOutWarps = 4, kOperandWarps = 8, kTma = kStateWarps + kOutWarps + kOperandWarps;
// Registers a thread: the state and output warps take what the others give up.  256 x 120 + 128 x 88 + 256 x 56 + 128 x 40 = the 768 x 80 of the launch.
constexpr int kLaunchRegs = 80, kStateRegs = 120, kOutRegs = 88, kOperandRegs = 56, kRestRegs = 40;
static_assert(256 * kStateRegs + 128 * kOutRegs + 256 * kOperandRegs + 128 * kRestRegs <= kThreads * kLaunchRegs, "no more than the launch had");
static_assert(kStateRegs > kLaunchRegs && kOutRegs > kLaunchRegs && kOperandRegs < kLaunchRegs && kRestRegs < kLaunchRegs, "up or down");

// Scalars of a chunk, 64 floats each: what it has decayed by up to a token, in the direction of time (units of log 2, in two parts), r, w,
// and f with the scale of the pairs.  Then the chunk's decay in two parts, and how many of its tokens are near its start.
enum { sUp = 0, sUpLo = 64, sRead = 128, sWrite = 192, sPair = 256, sDecay = 320, sNear = 322 };
// Tokens are near as long as no token in front of them has left this range: f, and what it scales, stay in the range of fp32 and bf16.
// One that is not has 2^(the whole part of its decay) taken into its row of x in front of the product with R (exact, or what is
// smaller than any number); its r has the rest, and its pairs' decays, against that whole part, are exponentials of their own.
// In a chunk with such tokens sPair holds the whole parts, 0 for near ones.
constexpr int kLeastNear = -96, kMostNear = 32;
// Inside the kernel R and what goes to it are in units of 2^24, and so is f: it is 2^(96 - 24) at most instead of 2^96, so that the pairs' sums
// stay numbers up to |x.y z| of 2^48 (2^24 without, behind a strong decay), while R and x.y keep both parts of what they are down to 2^-85.
// (Powers of two: no result in between changes by a bit.)
constexpr float kUnit = 16777216.f, kPerUnit = 1.f / kUnit;

struct Maps {
  CUtensorMap m[4], out[3];
};

// A bounded wait (tc::mbar_wait) as one short loop: every role has several, and what the roles run together in a chunk just fits
// the instruction cache.  (With the loops unrolled, operand by operand, 41 % of the backward's requests missed it, and a chunk took twice its time.)
__device__ __forceinline__ bool wait_phase(uint32_t bar, uint32_t parity) {
  uint32_t done;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t.reg .u32 n;\n\t"
      "mov.u32 n, %3;\n\t"
      "WAIT_%=:\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "@p bra.uni DONE_%=;\n\t"
      "sub.u32 n, n, 1;\n\t"
      "setp.ne.u32 q, n, 0;\n\t"
      "@q bra.uni WAIT_%=;\n\t"
      "DONE_%=:\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(done) : "r"(bar), "r"(parity), "n"(tc::kSpinLimit) : "memory");
  return done;
}

// 16 rows of an accumulator with M = 64, 16 columns, as mma.sync fragments (tmem_ld_rows).
__device__ __forceinline__ void load_rows16(uint32_t taddr, float (&v)[8]) {
  uint32_t* r = reinterpret_cast<uint32_t*>(v);
  asm volatile("tcgen05.ld.sync.aligned.16x256b.x2.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
               : "r"(taddr));
}

// Sums of four columns of two octets, 2 (lane % 4) and the next of each, over the eight lanes that hold them: every lane ends with one of
// them in v[0], two lanes with the same; returns which, less 2 (lane % 4).
__device__ __forceinline__ int column_sum(float (&v)[4], int lane) {
  const bool o = lane & 16, e = lane & 8;
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const float send = o ? v[k] : v[k + 2], keep = o ? v[k + 2] : v[k];
    v[k] = keep + __shfl_xor_sync(0xffffffffu, send, 16);
  }
  const float send = e ? v[0] : v[1], keep = e ? v[1] : v[0];
  v[0] = keep + __shfl_xor_sync(0xffffffffu, send, 8);
  v[0] += __shfl_xor_sync(0xffffffffu, v[0], 4);
  return (o ? 8 : 0) + (e ? 1 : 0);
}

__device__ __forceinline__ uint32_t times(uint32_t two, float by) {
  const float2 v = mul2(unpack_bf16(two), f2(by, by));
  return pack_bf16(v.x, v.y);
}
// Two values to a word of hi parts and one of lo parts, hi cut off instead of rounded: off by 2^-16 at most, for five instructions
// instead of seven.  For what ends in bf16 results alone.
__device__ __forceinline__ void split2_cut(float2 v, uint32_t& hi, uint32_t& lo) {
  const uint32_t a = __float_as_uint(v.x), b = __float_as_uint(v.y);
  hi = __byte_perm(a, b, 0x7632);
  const float2 r = fma2(f2(__uint_as_float(a & 0xffff0000u), __uint_as_float(b & 0xffff0000u)), f2(-1.f, -1.f), v);
  lo = pack_bf16(r.x, r.y);
}
// The same with hi rounded.
__device__ __forceinline__ void split2_round(float2 v, uint32_t& hi, uint32_t& lo) {
  hi = pack_bf16(v.x, v.y);
  const float2 r = fma2(f2(__uint_as_float(hi << 16), __uint_as_float(hi & 0xffff0000u)), f2(-1.f, -1.f), v);
  lo = pack_bf16(r.x, r.y);
}
__device__ __forceinline__ void stsm_x4_t(uint32_t addr, const uint32_t (&r)[4]) {
  asm volatile("stmatrix.sync.aligned.m8n8.x4.trans.shared.b16 [%0], {%1,%2,%3,%4};\n" ::"r"(addr), "r"(r[0]), "r"(r[1]), "r"(r[2]),
               "r"(r[3]) : "memory");
}
// A descriptor `bytes` further on (addresses of shared memory fill its low bits and do not overflow them).
__device__ __forceinline__ uint64_t step(uint64_t desc, uint32_t bytes) { return desc + (bytes >> 4); }

}  // namespace

// The decays of a row's pairs with two columns where not all tokens are near, against the whole part of the row's own (0 of a near row).
__device__ __forceinline__ float2 pair_decays(const float* sc, int row, int col, float scale) {
  const float whole = sc[sPair + row];
  return f2(scale * exp2f((whole - sc[sUp + col]) - sc[sUpLo + col]), scale * exp2f((whole - sc[sUp + col + 1]) - sc[sUpLo + col + 1]));
}

// What the gate's gradient takes of an operation (ChunkPass::reads, ::pairs) is compiled in: a CTA runs one of three bodies, each in one
// piece and without the others' branches, which would not fit the instruction cache together.
enum { kPlain, kReads, kPairs };
template <int D, int kKind>
__device__ __forceinline__ void walk_chunks(const Maps& maps, const ChunkCall& a, const int pi, const int block) {
  using C = Cfg<D>;
  constexpr int kStages = C::kStages;
  constexpr bool dots = kKind == kReads, sums = kKind == kPairs;
  extern __shared__ __align__(1024) unsigned char smem[];
  const int H = a.c.geo.heads;
  const Segments& sg = a.segments;
  const ChunkPass& t = a.pass[pi];
  const Pass& p = t.p;
  const bool rev = kept(p.reverse) != 0, walk = t.walk, states_only = kept(t.states_only) != 0;
  const int h = block % H;
  int n = block / H, seg = 0;
  if (walk && a.order) n = a.order[n];
  if (!walk && !find_segment(a.c.geo, sg, block / H, n, seg)) return;
  const SeqInfo sq = gdr::sequence(a.c.geo, n);
  const int all_segs = max((sq.nchunks + sg.chunks - 1) / sg.chunks, 1);
  if (states_only && seg == (rev ? 0 : all_segs - 1)) return;  // (nobody starts from it)
  const int c0 = seg * sg.chunks, c1 = walk ? sq.nchunks : min(c0 + sg.chunks, sq.nchunks);
  const int count = c1 - c0;
  const bool first_seg = walk || seg == (rev ? all_segs - 1 : 0), last_seg = walk || seg == (rev ? 0 : all_segs - 1);
  const size_t entry0 = (size_t)first_entry(a.c.geo, sg, n) * H + h;  // of the sequence's segments, H apart

  const int tid = threadIdx.x, warp = (int)tc::uniform(tid >> 5), lane = tid & 31;
  const int q = warp & 3, z = 32 * q + lane;  // this thread's channel of z
  const bool live = 32 * q < D;               // (heads of 64 channels fill half of the lanes; what the others hold goes nowhere)
  const uint32_t bars = smem_u32(smem), base = bars + C::kFront, slot = bars + 8 * C::bCount;
  unsigned char* tiles = smem + C::kFront;
  auto bar = [&](int b) { return bars + 8 * b; };
  if (warp == 0) tc::tmem_alloc(slot, C::kCols);
  if (tid == 32) {
    for (int s = 0; s < kStages; ++s) {
      tc::mbar_init(bar(C::bFull + s), 1);
      tc::mbar_init(bar(C::bEmpty + s), kOperandWarps + (states_only ? 1 : 2));     // who reads and writes them, the products of both warps
    }
    for (int s = 0; s < C::kRing; ++s) tc::mbar_init(bar(C::bScal + s), 1);
    for (int s = 0; s < 2; ++s) {
      for (int b : {(int)C::bU, (int)C::bKV, (int)C::bO, (int)C::bQK}) tc::mbar_init(bar(b + s), 1);
      for (int b : {(int)C::bQKfree, (int)C::bP, (int)C::bYw}) tc::mbar_init(bar(b + s), kOperandWarps);
      for (int b : {(int)C::bOut, (int)C::bOfree}) tc::mbar_init(bar(b + s), kOutWarps);
    }
    tc::mbar_init(bar(C::bQS), 1);
    for (int b : {(int)C::bR, (int)C::bKVfree}) tc::mbar_init(bar(b), kStateWarps);
    tc::fence_barrier_init();
  }
  tc::tc_fence_before();
  __syncthreads();
  launch_dependents();
  tc::tc_fence_after();
  const uint32_t tmem = tc::uniform(*reinterpret_cast<volatile uint32_t*>(smem + 8 * C::bCount));
  const uint32_t lanes = tmem + ((uint32_t)(32 * q) << 16);
  const size_t sbase = ((size_t)n * H + h) * D * D;
  auto entry = [&](int k) { return entry0 + (size_t)k * H; };
  bool ok = true;
  // Waits for phase `i` of a barrier (its i-th completion); all lanes of a warp together.
  auto wait = [&](int b, int i) {
    if (ok) ok = __all_sync(0xffffffffu, wait_phase(bar(b), i & 1));
  };
  // Of a pair of barriers, for even and for odd i, where i + 1 can complete before a waiter for i has looked: a barrier tells a phase
  // only from the next.
  auto wait2 = [&](int b, int i) { wait(b + (i & 1), i >> 1); };
  auto arrive = [&](int b) {  // one arrival a warp, after what its lanes did before
    __syncwarp();
    if (lane == 0) mbar_arrive(bar(b));
  };
  auto chunk = [&](int i) { return rev ? c1 - 1 - i : c0 + i; };
  auto valid_of = [&](int c) { return min(kChunk, sq.len - c * kChunk); };
  auto scalars = [&](int i) { return reinterpret_cast<float*>(tiles + C::oScal + (i % C::kRing) * C::kScal); };

  if (warp < kStateWarps) {
    tc::regs_up<kStateRegs>();
    // ------------------------------------------------------------------------------------------ the state
    constexpr int kS = D / 2;
    const int hf = warp >> 2, y0 = kS * hf;
    float S[kS];  // R[y0 + j][z] / kUnit
    float* const ends = kept(t.ends);
    float* const X = kept(t.X);
    // a state in memory, [y][z] or transposed
    auto load = [&](const float* from, bool transposed) {
#pragma unroll
      for (int j = 0; j < kS; j += 4) {
        if (!from || !live) {
          S[j] = S[j + 1] = S[j + 2] = S[j + 3] = 0.f;
        } else if (transposed) {
          const float4 x = __ldcg(reinterpret_cast<const float4*>(from + (size_t)z * D + y0 + j));
          S[j] = x.x * kPerUnit; S[j + 1] = x.y * kPerUnit; S[j + 2] = x.z * kPerUnit; S[j + 3] = x.w * kPerUnit;
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e) S[j + e] = __ldcg(from + (size_t)(y0 + j + e) * D + z) * kPerUnit;
        }
      }
    };
    auto store = [&](float* to, bool transposed) {
      if (!to || !live) return;
#pragma unroll
      for (int j = 0; j < kS; j += 4) {
        if (transposed) {
          *reinterpret_cast<float4*>(to + (size_t)z * D + y0 + j) = make_float4(S[j] * kUnit, S[j + 1] * kUnit, S[j + 2] * kUnit, S[j + 3] * kUnit);
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e) to[(size_t)(y0 + j + e) * D + z] = S[j + e] * kUnit;
        }
      }
    };
    if (states_only) load(nullptr, false);
    else load(first_seg ? (p.init ? p.init + sbase : nullptr) : t.starts + entry(seg + (rev ? 1 : -1)) * D * D, p.init_t);
    for (int i = 0; i < count && ok; ++i) {
      const int c = chunk(i), cs = c / sg.chunks;
      if (X && (i == 0 || (c + 1) % sg.chunks == 0)) {  // <state, R> at the end of segment cs; [z][y] is the state's order here
        float x = 0.f;
        if (live) {
          const float* s = t.X_states + entry(cs) * D * D + (size_t)z * D + y0;
#pragma unroll
          for (int j = 0; j < kS; j += 4) {
            const float4 v = __ldcg(reinterpret_cast<const float4*>(s + j));
            x = fmaf(v.x, S[j], fmaf(v.y, S[j + 1], fmaf(v.z, S[j + 2], fmaf(v.w, S[j + 3], x))));
          }
        }
#pragma unroll
        for (int o = 16; o; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
        if (lane == 0) X[entry(cs) * kXParts + warp] = x * kUnit;
      }
      if (!states_only) {
        if (i > 0) wait(C::bQS, i - 1);  // the reads of the chunk before are done with R's operand
        if (!ok) break;
        if (live) {
#pragma unroll
          for (int g = 0; g < kS / 32; ++g) {
            uint32_t hi[16], lo[16];
#pragma unroll
            for (int j = 0; j < 16; ++j) split2_round(f2(S[32 * g + 2 * j], S[32 * g + 2 * j + 1]), hi[j], lo[j]);
            tc::tmem_st16(lanes + C::cR + kS / 2 * hf + 16 * g, hi);
            tc::tmem_st16(lanes + C::cR + kS + kS / 2 * hf + 16 * g, lo);
          }
          tc::tmem_st_wait();
        }
        tc::tc_fence_before();
        arrive(C::bR);
      }
      wait(C::bScal + i % C::kRing, i / C::kRing);
      if (!ok) break;
      const float2 dec = *reinterpret_cast<const float2*>(scalars(i) + sDecay);
      wait2(C::bKV, i);
      if (!ok) break;
      tc::tc_fence_after();
      if (live) {
        const float2 dh = f2(dec.x, dec.x), dl = f2(dec.y, dec.y);
#pragma unroll
        for (int part = 0; part < kS / 32; ++part) {
          float x[32];
          tc::tmem_ld32(lanes + C::cKV + y0 + 32 * part, x);
          tc::tmem_ld_wait();
          if (part == kS / 32 - 1) {
            tc::tc_fence_before();
            arrive(C::bKVfree);
          }
#pragma unroll
          for (int j = 0; j < 32; j += 2) {
            float* s = S + 32 * part + j;
            const float2 r = fma2(f2(s[0], s[1]), dh, fma2(f2(s[0], s[1]), dl, f2(x[j], x[j + 1])));
            s[0] = r.x;
            s[1] = r.y;
          }
        }
      } else {
        tc::tc_fence_before();
        arrive(C::bKVfree);
      }
      const bool end = i == count - 1 || (rev ? c % sg.chunks == 0 : (c + 1) % sg.chunks == 0);
      if (end && ends && (walk || states_only || last_seg)) store(ends + entry(cs) * D * D, p.fin_t);
    }
    if (!ok) {
      if (lane == 0) atomicExch(a.status, 1);
    } else if (last_seg) {
      store(p.fin ? p.fin + sbase : nullptr, p.fin_t);
    }
  } else if (warp < kStateWarps + kOutWarps) {
    tc::regs_up<kOutRegs>();
    // ------------------------------------------------------------------------------------------ the output
    // A warp reads its accumulators as 8 x 8 matrices (16 lanes at a time), tokens along a row: transposed by stmatrix they are rows of
    // channels in the place of the chunk's u, which they have read by then, and leave from there.
    const int count_out = states_only ? 0 : count;
    const int t2 = 2 * (lane & 3);
    float* const dot_to = kept(p.dots + ((size_t)q * H + h) * a.c.geo.total_tokens + t2);
    float* const out32 = kept(p.out32 ? static_cast<float*>(p.out) + (size_t)h * D + 32 * q + (lane >> 2) : nullptr);
    const int row32 = kept(H * D);
    // the row whose address this lane gives to stmatrix and ldmatrix: token lane % 8 of an octet, channels 8 (lane / 8) .. of the warp's
    const uint32_t at = (q >> 1) * 8192 + (lane & 7) * 128 + (((4 * (q & 1) + (lane >> 3)) ^ (lane & 7)) << 4);
    auto output = [&](auto in_fp32) {  // (one or the other for all of the CTA's chunks)
      constexpr bool kDots = dots, k32 = decltype(in_fp32)::value;
      for (int i = 0; i < count_out && ok; ++i) {
        const int c = chunk(i), valid = valid_of(c), tok0 = sq.bos + c * kChunk;
        const float* r = scalars(i) + sRead + t2;
        wait(C::bScal + i % C::kRing, i / C::kRing);
        wait2(C::bO, i);
        wait2(C::bU, i);  // (u, and so that the slot is free)
        if (!ok) break;
        tc::tc_fence_after();
        uint32_t slot_at = base + C::oU + (i & 1) * C::kTile + at;
        if (live) {
          // (Rolled, here and below: every warp runs its code once a chunk, and all of it together has to stay in the instruction cache.)
          uint32_t acc = lanes + (!(i & 1) ? C::cO : kDots ? C::cW : C::cO + 64), pv_at = lanes + C::cO + 64;
#pragma unroll 1
          for (int part = 0; part < 4; ++part) {  // two octets of tokens
            float x[2][8], y[2][8], dot[4];
#pragma unroll
            for (int m = 0; m < 2; ++m) {
              load_rows16(acc + ((uint32_t)(16 * m) << 16), x[m]);
              if (kDots) load_rows16(pv_at + ((uint32_t)(16 * m) << 16), y[m]);
            }
            uint32_t uu[2][4];
            float2 rr[2];
#pragma unroll
            for (int o = 0; o < 2; ++o) {
              rr[o] = *reinterpret_cast<const float2*>(r + 8 * o);
              if (kDots) ldsm_x4_t(uu[o], slot_at + o * 1024);
            }
            tc::tmem_ld_wait();
#pragma unroll
            for (int o = 0; o < 2; ++o) {
              uint32_t out[4];
              float2 sum = f2(0.f, 0.f);
#pragma unroll
              for (int m = 0; m < 4; ++m) {  // channels 8 m + lane / 4
                const int e = 4 * o + 2 * (m & 1);
                float2 v = mul2(f2(x[m >> 1][e], x[m >> 1][e + 1]), rr[o]);
                if (kDots) {
                  sum = fma2(v, unpack_bf16(uu[o][m]), sum);
                  v = fma2(f2(y[m >> 1][e], y[m >> 1][e + 1]), rr[o], v);
                }
                if (k32) {
                  const int tk = 16 * part + 8 * o + t2;
                  float* to = out32 + (size_t)(tok0 + tk) * row32 + 8 * m;
                  if (tk < valid) to[0] = v.x;
                  if (tk + 1 < valid) to[row32] = v.y;
                } else {
                  out[m] = pack_bf16(v.x, v.y);
                }
              }
              dot[2 * o] = sum.x;
              dot[2 * o + 1] = sum.y;
              if (!k32) stsm_x4_t(slot_at + o * 1024, out);
            }
            if (kDots) {
              const int tk = 16 * part + column_sum(dot, lane);
              if (tk + t2 < valid) dot_to[tok0 + tk] = dot[0];
            }
            acc += 16;
            pv_at += 16;
            slot_at += 2048;
            r += 16;
          }
        }
        tc::tc_fence_before();
        arrive(C::bOfree + (i & 1));
        tc::fence_proxy_async();
        arrive(C::bOut + (i & 1));
      }
    };
    if (out32) output(std::integral_constant<bool, true>{}); else output(std::integral_constant<bool, false>{});
    if (!ok && lane == 0) atomicExch(a.status, 1);
  } else if (warp < kTma) {
    tc::regs_down<kOperandRegs>();
    // ------------------------------------------------------------------------------------------ weighted keys and pairs
    const int hf = (warp - kStateWarps - kOutWarps) >> 2, me = 128 * hf + 32 * q + lane;
    const int row = 16 * q + (lane >> 2), col2 = 2 * (lane & 3);
    float* const dots_of = kept(p.dots + (size_t)h * a.c.geo.total_tokens);
    const float pair_scale = kept((rev ? p.c : 1.f) * kPerUnit);  // (c / read)
    const int sign_of = kept(rev ? -1 : 1);
    const bool qk_in_turn = !sums && !dots;
    // the row whose address this lane gives to stmatrix: rows 8 (m & 1) .. of octet m >> 1
    const uint32_t to = base + C::oP + ((lane >> 4) & 1) * 1024 + (16 * q + 8 * ((lane >> 3) & 1) + (lane & 7)) * 16;
    // pieces of 16 bytes: token (me >> 3) + 32 j, each in its swizzled place
    const uint32_t piece = (me >> 3) * 128 + (me & 7) * 16;
    // P has zeros where no pair is, for good: a warp's own rows of the blocks that are its own.
    for (int e = lane; e < 8 * 16; e += 32) {
      const int octet = 2 * (hf + (e >> 6) * 2) + ((e >> 4) & 1), part = (e >> 5) & 1;
      *reinterpret_cast<uint4*>(tiles + C::oP + part * 8192 + octet * 1024 + (16 * q + (e & 15)) * 16) = make_uint4(0, 0, 0, 0);
    }
    __syncwarp();
    {
      constexpr bool kSums = sums;
      for (int i = 0; i < count && ok; ++i) {
        const int c = chunk(i), valid = valid_of(c), tok0 = sq.bos + c * kChunk;
        const float* sc = scalars(i);
        wait(C::bFull + i % kStages, i / kStages);
        wait(C::bScal + i % C::kRing, i / C::kRing);
        if (!states_only) wait2(C::bQK, i);  // (the pairs have read the keys, whose place is taken)
        if (i > 0) wait2(C::bKV, i - 1);    // the product with what is in the buffer is done
        if (!ok) break;
        {
          unsigned char* y = tiles + (i % kStages) * C::kStage + C::oY + piece;
          unsigned char* ylo = tiles + C::oYlo + piece;
#pragma unroll 1
          for (int j = 0; j < D / 32; ++j) {  // half a block of 64 channels a turn
            const uint32_t at = (j >> 1) * 8192 + (j & 1) * 4096;
            const int tk = (me >> 3) + 32 * (j & 1);
            const uint4 v = *reinterpret_cast<const uint4*>(y + at);
            const float f = tk < valid ? sc[sWrite + tk] : 0.f;
            const float2 ff = f2(f, f);
            uint4 hi, lo;
            split2_round(mul2(unpack_bf16(v.x), ff), hi.x, lo.x);
            split2_round(mul2(unpack_bf16(v.y), ff), hi.y, lo.y);
            split2_round(mul2(unpack_bf16(v.z), ff), hi.z, lo.z);
            split2_round(mul2(unpack_bf16(v.w), ff), hi.w, lo.w);
            if (tk >= valid) hi = lo = make_uint4(0, 0, 0, 0);
            *reinterpret_cast<uint4*>(y + at) = hi;
            *reinterpret_cast<uint4*>(ylo + at) = lo;
          }
        }
        const int near = states_only ? kChunk : (int)sc[sNear];
        if (near < kChunk) {  // (the pairs have read x)
          unsigned char* x = tiles + (i % kStages) * C::kStage + C::oX + piece;
#pragma unroll 1
          for (int j = 0; j < D / 32; ++j) {
            const int tk = (me >> 3) + 32 * (j & 1);
            if ((rev ? kChunk - 1 - tk : tk) < near) continue;
            uint4* const at = reinterpret_cast<uint4*>(x + (j >> 1) * 8192 + (j & 1) * 4096);
            const float up = __int_as_float(min(max((int)sc[sPair + tk] + 127, 0), 255) << 23);  // (0 below 2^-126, infinity from 2^128 on)
            uint4 v = *at;
            v.x = times(v.x, up);
            v.y = times(v.y, up);
            v.z = times(v.z, up);
            v.w = times(v.w, up);
            *at = v;
          }
        }
        tc::fence_proxy_async();
        arrive(C::bYw + (i & 1));
        if (states_only) {
          arrive(C::bEmpty + i % kStages);  // (what was loaded has been stored)
          continue;
        }
        if (i > 0) wait2(C::bO, i - 1);  // (as above)
        if (!ok) break;
        tc::tc_fence_after();
        // Blocks of 16 columns against the warp's 16 rows: those in front of the diagonal (in the direction of time) are whole, its own is
        // masked, the others have no pairs.  Two at most are this warp's.
        float rows[2] = {0.f, 0.f};
        float* dot = dots_of + tok0;
        const size_t slice = (size_t)H * a.c.geo.total_tokens;
        uint32_t seen = 0;
#pragma unroll 1
        for (int blk = hf; blk < 4; blk += 2) {
          const int rel = rev ? blk - q : q - blk;
          if (rel < 0) {
            if (kSums && 16 * blk + (lane >> 1) < valid) dot[q * slice + 16 * blk + (lane >> 1)] = 0.f;
            continue;
          }
          float x[8], w[8], cols[4];
          load_rows16(lanes + (qk_in_turn && (i & 1) ? C::cW : C::cQK) + 16 * blk, x);
          if (kSums) load_rows16(lanes + C::cW + 16 * blk, w);
          tc::tmem_ld_wait();
          uint32_t hi[4], lo[4];
          const int whole = rel > 0 ? kChunk : 0;
#pragma unroll
          for (int o = 0; o < 2; ++o) {
            const int col = 16 * blk + 8 * o + col2;
            float2 f0, f1;  // of the two rows
            if (near == kChunk) {
              f0 = f1 = *reinterpret_cast<const float2*>(sc + sPair + col);
            } else {
              f0 = pair_decays(sc, row, col, pair_scale);
              f1 = pair_decays(sc, row + 8, col, pair_scale);
            }
            float2 v[2] = {mul2(f2(x[4 * o], x[4 * o + 1]), f0), mul2(f2(x[4 * o + 2], x[4 * o + 3]), f1)};
            const int d = sign_of * (row - col) + whole;  // on the diagonal 0
            v[0].x = d >= 0 ? v[0].x : 0.f;
            v[0].y = d >= sign_of ? v[0].y : 0.f;
            v[1].x = d >= -8 * sign_of ? v[1].x : 0.f;
            v[1].y = d >= -7 * sign_of ? v[1].y : 0.f;
            split2_cut(v[0], hi[2 * o], lo[2 * o]);
            split2_cut(v[1], hi[2 * o + 1], lo[2 * o + 1]);
            if (kSums) {  // (a token's own pair has no decay in it)
              const float r0 = sc[sRead + row], r1 = sc[sRead + row + 8];
              float2 s0 = mul2(mul2(v[0], f2(r0, r0)), f2(w[4 * o], w[4 * o + 1]));
              float2 s1 = mul2(mul2(v[1], f2(r1, r1)), f2(w[4 * o + 2], w[4 * o + 3]));
              s0.x = d > 0 ? s0.x : 0.f;
              s0.y = d > sign_of ? s0.y : 0.f;
              s1.x = d > -8 * sign_of ? s1.x : 0.f;
              s1.y = d > -7 * sign_of ? s1.y : 0.f;
              rows[0] += s0.x + s0.y;
              rows[1] += s1.x + s1.y;
              cols[2 * o] = s0.x + s1.x;
              cols[2 * o + 1] = s0.y + s1.y;
            }
          }
          stsm_x4(to + 2048 * blk, hi);
          stsm_x4(to + 8192 + 2048 * blk, lo);
          seen ^= hi[0] ^ hi[1] ^ hi[2] ^ hi[3];
          if (kSums) {
            const int col = 16 * blk + column_sum(cols, lane) + col2;
            if (col < valid) dot[q * slice + col] = -cols[0];
          }
        }
        tc::tc_fence_before();
        arrive(C::bQKfree + (i & 1));
        tc::fence_proxy_async();
        arrive(C::bP + (i & 1));
        arrive_behind_loads(bar(C::bEmpty + i % kStages), seen);
        if (kSums) {
#pragma unroll
          for (int o = 1; o < 4; o <<= 1) {
            rows[0] += __shfl_xor_sync(0xffffffffu, rows[0], o);
            rows[1] += __shfl_xor_sync(0xffffffffu, rows[1], o);
          }
          if ((lane & 3) < 2) {
            const int tk = row + 8 * (lane & 3);
            if (tk < valid) dot[(4 + hf) * slice + tk] = lane & 1 ? rows[1] : rows[0];
          }
        }
      }
    }
    if (!ok && lane == 0) atomicExch(a.status, 1);
  } else {
    tc::regs_down<kRestRegs>();
    if (warp == kTma) {
      // ------------------------------------------------------------------------------------------ tiles and scalars
      const int hx = kept(h / p.x_group), hy = kept(h / p.y_group), hz = kept(h / p.z_group);
      const CUtensorMap *mx = kept(&maps.m[t.map[0]]), *my = kept(&maps.m[t.map[1]]), *mz = kept(&maps.m[t.map[2]]);
      const float read = kept(p.read * kUnit), write = kept(p.write * kPerUnit), pair_scale = kept((rev ? p.c : 1.f) * kPerUnit);
      int asked = 0;  // chunks whose tiles have been asked for
      // Lane l owns tokens l and l + 32.  The scalars go a chunk in front of the tiles.
      auto gates = [&](int i, float (&g)[2]) {
        const int c = chunk(min(i, count - 1)), valid = valid_of(c);
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int tk = lane + 32 * e;
          g[e] = tk < valid ? gate(a.c, (size_t)(sq.bos + c * kChunk + tk), h) : 0.f;
        }
      };
      float next[2] = {0.f, 0.f};
      unsigned long long total = 0;  // (asked for of single segments alone; a long walk's may wrap)
      // Backwards: a segment's first chunk is the last one of it that comes.
      int* grows_at = dots && t.grows && count > 0 ? t.grows + entry((c1 - 1) / sg.chunks) : nullptr;
      int to_go = dots && count > 0 ? (c1 - 1) % sg.chunks : 0;
      float top = 0.f;
      auto scalars_of = [&](int i) {
        const bool bad = __any_sync(0xffffffffu, next[0] != next[0] || next[1] != next[1]);
        if (dots && grows_at) {
          top = fmaxf(top, fmaxf(next[0], next[1]));
          if (--to_go < 0) {
            const int grows = __any_sync(0xffffffffu, top > 0.f);
            if (lane == 0) *grows_at = grows;
            top = 0.f;
            grows_at -= H;
            to_go = sg.chunks - 1;
          }
        }
        long long run[2] = {to_fixed(next[0]), to_fixed(next[1])};
        gates(i + 1, next);
#pragma unroll 1
        for (int o = 1; o < 32; o <<= 1) {
          const long long y0 = __shfl_up_sync(0xffffffffu, run[0], o), y1 = __shfl_up_sync(0xffffffffu, run[1], o);
          if (lane >= o) {
            run[0] += y0;
            run[1] += y1;
          }
        }
        run[1] += __shfl_sync(0xffffffffu, run[0], 31);
        const long long GL = __shfl_sync(0xffffffffu, run[1], 31);
        total += GL;
        float2 dec = exp2_fixed_two(GL);
        const float none = bad ? __int_as_float(0x7fc00000) : 1.f;  // (a gate that is no number makes none of its chunk's results one)
        float* out = scalars(i) + lane;
        if (rev) {  // the chunk's decay up to each token, in the direction of time
          run[0] = GL - run[0];
          run[1] = GL - run[1];
        }
        auto leaves = [&](long long up) {
          const int w = (int)(up >> kFixed);
          return __ballot_sync(0xffffffffu, w < kLeastNear || w >= kMostNear);
        };
        const unsigned far0 = leaves(run[0]), far1 = leaves(run[1]);  // tokens 0..31 and 32..63
        const int near = rev ? (far1 ? __clz(far1) : 32 + __clz(far0)) : far0 ? __ffs(far0) - 1 : far1 ? 31 + __ffs(far1) : kChunk;
#pragma unroll 1
        for (int e = 0; e < 2; ++e) {
          const long long up = e ? run[1] : run[0];
          out[sWrite] = write * exp2_fixed(GL - up) * none;
          if (!states_only) {
            const int tk = lane + 32 * e, whole = (rev ? kChunk - 1 - tk : tk) < near ? 0 : (int)(up >> kFixed);
            const float2 two = from_fixed(up);
            out[sUp] = two.x * none;
            out[sUpLo] = two.y;
            out[sRead] = read * exp2_fixed(up - ((long long)whole << kFixed)) * none;
            out[sPair] = near < kChunk ? (float)whole : pair_scale * exp2_fixed(-up) * none;
          }
          out += 32;
        }
        if (lane == 0) {
          out = scalars(i);
          out[sDecay] = dec.x * none;
          out[sDecay + 1] = dec.y;
          out[sNear] = (float)near;
        }
        arrive(C::bScal + i % C::kRing);
      };
      if (count > 0) {
        gates(0, next);
        scalars_of(0);
      }
      for (int i = 0; i < count && ok; ++i) {
        if (i >= kStages) wait(C::bEmpty + i % kStages, i / kStages - 1);
        if (!ok) break;
        if (lane == 0) {
          const int tok0 = sq.bos + chunk(i) * kChunk;
          const uint32_t st = base + (i % kStages) * C::kStage, full = bar(C::bFull + i % kStages);
          tc::mbar_expect_tx(full, (states_only ? 2 : 3) * C::kTile);
#pragma unroll
          for (int b = 0; b < D / 64; ++b) tc::tma_load_3d(st + C::oY + 8192 * b, my, full, 64 * b, hy, tok0);
#pragma unroll
          for (int b = 0; b < D / 64; ++b) tc::tma_load_3d(st + C::oZ + 8192 * b, mz, full, 64 * b, hz, tok0);
          if (!states_only) {
#pragma unroll
            for (int b = 0; b < D / 64; ++b) tc::tma_load_3d(st + C::oX + 8192 * b, mx, full, 64 * b, hx, tok0);
          }
        }
        asked = i + 1;
        __syncwarp();
        if (i + 1 < count) scalars_of(i + 1);
      }
      if (!ok && lane == 0) {
        atomicExch(a.status, 1);
        // copies in flight have to land before the CTA's shared memory goes to another
        for (int j = asked > kStages ? asked - kStages : 0; j < asked; ++j) tc::mbar_wait(bar(C::bFull + j % kStages), (j / kStages) & 1);
      }
      if (states_only && lane == 0) t.decay[entry(seg)] = (double)(long long)total * (1.0 / (1ll << kFixed));
    } else if (warp <= kTma + 2) {
      constexpr uint32_t qk = tc::idesc_bf16(64, 64, false, false), pv = tc::idesc_bf16(128, 64, true, false),
                         qs = tc::idesc_bf16(128, 64, false, false), kv = tc::idesc_bf16(128, D, true, true);
      auto stage = [&](int i) { return tc::uniform(base + (i % kStages) * C::kStage); };  // (descriptors in uniform registers: pkda_tc.cuh)
      // `outer` times four products of 16 of K, operands `sa`, `sb` bytes on with each; the next four start `oa`, `ob` bytes on.
      auto products = [&](uint32_t acc, uint64_t da, uint64_t db, uint32_t idesc, int outer, uint32_t sa, uint32_t sb, int oa, int ob,
                          bool onto = false) {
#pragma unroll 1
        for (int k = 0; k < outer; ++k) {
#pragma unroll
          for (int kk = 0; kk < 4; ++kk) tc::umma_bf16(acc, step(da, kk * sa), step(db, kk * sb), idesc, onto || k > 0 || kk > 0);
          da += (long long)(oa >> 4);
          db += (long long)(ob >> 4);
        }
      };
      if (warp == kTma + 1) {
        // ---------------------------------------------------------------------------------------- products of the inputs: x y^T and KV
        const bool two = !sums && !dots;  // two accumulators take turns where there is room
        auto pairs = [&](int i) {  // the tiles of chunk i are here: its x y^T
          const uint64_t x = tc::desc_kmajor(stage(i)), u = tc::desc_kmajor(tc::uniform(base + C::oU + (i & 1) * C::kTile));
          if (tc::elect_one()) {
            products(tmem + (two && (i & 1) ? C::cW : C::cQK), step(x, C::oX), step(x, C::oY), qk, D / 64, 32, 32, 8192, 8192);
            if (sums) products(tmem + C::cW, u, step(x, C::oZ), qk, D / 64, 32, 32, 8192, 8192);
            tc::umma_commit(bar(C::bQK + (i & 1)));
          }
          __syncwarp();
        };
        auto arrived = [&](int i) {
          wait(C::bFull + i % kStages, i / kStages);
          const int valid = valid_of(chunk(i));
          if (ok && valid < kChunk) {  // (the next sequence's tokens: zero times a NaN of theirs would not be zero)
            unsigned char* rows = tiles + (i % kStages) * C::kStage;
            for (int e = lane; e < (kChunk - valid) * (D / 8); e += 32) {
              const int tk = valid + e / (D / 8), piece = e % (D / 8);
              const uint32_t at = (piece >> 3) * 8192 + tk * 128 + ((piece & 7) << 4);
              *reinterpret_cast<uint4*>(rows + C::oZ + at) = make_uint4(0, 0, 0, 0);
              if (!states_only) *reinterpret_cast<uint4*>(rows + C::oY + at) = make_uint4(0, 0, 0, 0);
            }
            tc::fence_proxy_async();
            __syncwarp();
          }
        };
        auto ready = [&](int b, int i) { return __all_sync(0xffffffffu, tc::mbar_test(bar(b), i & 1)); };
        int asked = 0;  // chunks whose tiles have been waited for and whose pairs are under way
        auto ask = [&]() {
          arrived(asked);
          if (!states_only) {
            if (asked > two) wait2(C::bQKfree, asked - 1 - two);
            if (sums) wait2(C::bU, asked);
            if (!ok) return;
            tc::tc_fence_after();
            pairs(asked);
          }
          ++asked;
        };
        // The pairs of the next chunk wait for none of this one's, and much waits for them: in front of whatever comes, when they can.
        auto try_ask = [&](int next) {
          if (ok && asked == next && next < count && ready(C::bFull + next % kStages, next / kStages) &&
              (next <= two || ready(C::bQKfree + ((next - 1 - two) & 1), (next - 1 - two) >> 1)) &&
              (!sums || ready(C::bU + (next & 1), next >> 1)))
            ask();
        };
        auto wait_asking = [&](int b, int i, int next) {
          for (uint32_t it = 0; ok && it < tc::kSpinLimit; ++it) {
            try_ask(next);
            if (asked != next || next >= count) return wait(b, i);
            if (ready(b, i)) return;
          }
          ok = false;
        };
        for (int i = 0; i < count && ok; ++i) {
          const uint32_t st = stage(i);
          if (asked == i) ask();
          if (!ok) break;
          wait_asking(C::bYw + (i & 1), i >> 1, i + 1);
          if (i > 0) wait(C::bKVfree, i - 1);
          if (!ok) break;
          tc::tc_fence_after();
          const uint64_t tile = tc::desc_mnmajor(st, 8192), z = step(tile, C::oZ), yhi = step(tile, C::oY);
          const uint64_t ylo = tc::desc_mnmajor(base + C::oYlo, 8192);
          if (tc::elect_one()) {
#pragma unroll 1
            for (int k = 0; k < 2; ++k) {
              const uint64_t y = k ? ylo : yhi;
#pragma unroll
              for (int kk = 0; kk < 4; ++kk) tc::umma_bf16(tmem + C::cKV, step(z, kk * 2048), step(y, kk * 2048), kv, k > 0 || kk > 0);
            }
            tc::umma_commit(bar(C::bKV + (i & 1)));
            tc::umma_commit(bar(C::bEmpty + i % kStages));
          }
          __syncwarp();
        }
      } else if (!states_only) {
        // ---------------------------------------------------------------------------------------- products with the state and with P
        for (int i = 0; i < count && ok; ++i) {
          const uint32_t st = stage(i);
          wait(C::bR, i);
          if (!dots && i > 1) wait2(C::bOfree, i - 2);
          wait(C::bFull + i % kStages, i / kStages);
          wait(C::bScal + i % C::kRing, i / C::kRing);
          if (!ok) break;
          const bool cut = __any_sync(0xffffffffu, scalars(i)[sNear] < kChunk);
          if (cut) wait2(C::bP, i);  // (whoever leaves P has changed rows of x before)
          if (!ok) break;
          tc::tc_fence_after();
          const uint64_t x = step(tc::desc_kmajor(st), C::oX);
          const uint32_t out = tmem + (!(i & 1) ? C::cO : dots ? C::cW : C::cO + 64);
          if (tc::elect_one()) {
#pragma unroll 1
            for (int k = 0; k < D / 32; ++k) {  // hi and lo, 64 of K each
              const uint64_t xb = step(x, (k & (D / 64 - 1)) * 8192);
#pragma unroll
              for (int kk = 0; kk < 4; ++kk) tc::umma_bf16_ta(out, tmem + C::cR + 32 * k + 8 * kk, step(xb, kk * 32), qs, k > 0 || kk > 0);
            }
            tc::umma_commit(bar(C::bQS));
          }
          __syncwarp();
          if (!cut) wait2(C::bP, i);
          if (dots && i > 0) wait2(C::bOfree, i - 1);  // (PV has one accumulator then)
          if (!ok) break;
          tc::tc_fence_after();
          const uint64_t pairs_at = gdr::pair_desc(base + C::oP, 0);
          if (tc::elect_one()) {
            products(dots ? tmem + C::cO + 64 : out, step(tc::desc_mnmajor(st, 8192), C::oZ), pairs_at, pv, 2, 2048, 2048, 0, 8192, !dots);
            tc::umma_commit(bar(C::bO + (i & 1)));
            tc::umma_commit(bar(C::bEmpty + i % kStages));
          }
          __syncwarp();
        }
      }
      if (!ok && lane == 0) atomicExch(a.status, 1);
    } else {
      // ------------------------------------------------------------------------------------------ u in, results out
      const int count_out = states_only ? 0 : count;
      const bool reads_u = dots || sums;
      const int hu = kept(reads_u ? h / p.u_group : 0);
      const CUtensorMap *mu = kept(&maps.m[t.map[3]]), *mo = kept(&maps.out[pi]);
      bf16* const out = kept(p.out32 ? nullptr : static_cast<bf16*>(p.out));
      auto open = [&](int i) {  // the slot of chunk i: u comes, or it is free at once
        if (i >= count_out || lane != 0) return;
        if (reads_u) {
          const uint32_t at = base + C::oU + (i & 1) * C::kTile;
          tc::mbar_expect_tx(bar(C::bU + (i & 1)), C::kTile);
#pragma unroll
          for (int b = 0; b < D / 64; ++b)
            tc::tma_load_3d(at + 8192 * b, mu, bar(C::bU + (i & 1)), 64 * b, hu, sq.bos + chunk(i) * kChunk);
        } else {
          mbar_arrive(bar(C::bU + (i & 1)));
        }
      };
      open(0);
      open(1);
      int i = 0;
      for (; i < count_out && ok; ++i) {
        const int c = chunk(i), valid = valid_of(c), tok0 = sq.bos + c * kChunk;
        wait2(C::bOut, i);
        if (!ok) break;
        if (out) {
          if (valid == kChunk) {
            if (lane == 0) {
#pragma unroll
              for (int b = 0; b < D / 64; ++b)
                tc::tma_store_3d(mo, base + C::oU + (i & 1) * C::kTile + 8192 * b, 64 * b, h, tok0);
              tc::bulk_commit();
              tc::bulk_wait_read();
            }
          } else {  // (what lies behind the sequence is not ours)
            const unsigned char* x = tiles + C::oU + (i & 1) * C::kTile;
            for (int e = lane; e < valid * (D / 8); e += 32) {
              const int tk = e / (D / 8), pc = e % (D / 8);
              *reinterpret_cast<uint4*>(out + ((size_t)(tok0 + tk) * H + h) * D + 8 * pc) =
                  *reinterpret_cast<const uint4*>(x + (pc >> 3) * 8192 + tk * 128 + (((pc & 7) ^ (tk & 7)) << 4));
            }
          }
        }
        __syncwarp();
        open(i + 2);
      }
      if (lane == 0) tc::bulk_wait_all();  // (it must have left before the CTA's shared memory goes to another)
      if (!ok && lane == 0) {
        atomicExch(a.status, 1);
        for (int j = i; j < min(i + 2, count_out); ++j) tc::mbar_wait(bar(C::bU + (j & 1)), (j >> 1) & 1);  // (copies in flight have to land)
      }
    }
  }
  tc::tc_fence_before();
  __syncthreads();
  if (warp == 0) tc::tmem_dealloc(tmem, C::kCols);
  // If any kernel of the call gave up (this CTA included), the first output row of this CTA and its states become NaN, so that a
  // caller who never reads the status word cannot take a partial result for a complete one.
  if (warp == 1 && *reinterpret_cast<volatile int*>(a.status) != 0) {
    const size_t at = ((size_t)(sq.bos + c0 * kChunk) * H + h) * D;
    if (p.out && count > 0) {
      if (p.out32) mark_failed(static_cast<float*>(p.out) + at, D);
      else mark_failed(static_cast<bf16*>(p.out) + at, D);
    }
    if (p.dots && count > 0 && lane == 0) p.dots[(size_t)h * a.c.geo.total_tokens + sq.bos + c0 * kChunk] = __int_as_float(0x7fc00000);
    if (p.fin && last_seg) mark_failed(p.fin + sbase, D * D);
  }
}

template <int D>
__global__ void __launch_bounds__(kThreads, 1) la_chunk_kernel(const __grid_constant__ Maps maps, const __grid_constant__ ChunkCall a) {
  wait_prerequisites();
  // Which operation, and which of its sequences, heads and segments.  One operation behind the other: SMs next to one another share an
  // instruction cache, and two of the bodies do not fit it (8 x 4,096 tokens of 16 heads, dv beside dk: 4.8 and 5.6 us a chunk instead of 2.8).
  int block = blockIdx.x, pi = 0;
  for (; pi + 1 < a.n; ++pi) {
    const int n = a.c.geo.heads * (a.pass[pi].walk ? a.c.geo.n_seqs : (int)a.segments.entries);
    if (block < n) break;
    block -= n;
  }
  if (a.pass[pi].reads) walk_chunks<D, kReads>(maps, a, pi, block);
  else if (a.pass[pi].pairs) walk_chunks<D, kPairs>(maps, a, pi, block);
  else walk_chunks<D, kPlain>(maps, a, pi, block);
}

// Tensor map of a [tokens][heads][D] activation in boxes of 64 channels x 64 tokens of one head.
static bool map_rows(CUtensorMap* m, const void* base, int heads, int tokens, int D) {
  const uint64_t dims[3] = {(uint64_t)D, (uint64_t)heads, (uint64_t)tokens}, str[2] = {(uint64_t)D * 2, (uint64_t)heads * D * 2};
  const uint32_t box[3] = {64, 1, 64};
  return encode_bf16_map(m, base, 3, dims, str, box);
}

template <int D> static int launch(const ChunkCall& a, const Maps& maps, int grid, cudaStream_t st) {
  const auto kernel = la_chunk_kernel<D>;
  if (!ensure_dynamic_smem(kernel, Cfg<D>::kSmem)) return PKDA_ERR_LAUNCH;
  begin_stage(a.pass[0].states_only ? kStageLaStates : kStageLaChunks, st);
  const int rc = launch_kernel(kernel, grid, kThreads, Cfg<D>::kSmem, st, maps, a);
  end_stage(st);
  return rc;
}

int launch_chunks(const ChunkCall& a, cudaStream_t st) {
  Maps maps;
  for (int i = 0; i < 4; ++i)
    if (a.base[i] && !map_rows(&maps.m[i], a.base[i], a.heads[i], a.c.geo.total_tokens, a.D)) return PKDA_ERR_LAUNCH;
  for (int i = 0; i < a.n; ++i) {
    const Pass& p = a.pass[i].p;
    if (p.out && !p.out32 && !map_rows(&maps.out[i], p.out, a.c.geo.heads, a.c.geo.total_tokens, a.D)) return PKDA_ERR_LAUNCH;
  }
  long long grid = 0;
  for (int i = 0; i < a.n; ++i) grid += a.c.geo.heads * (a.pass[i].walk ? a.c.geo.n_seqs : a.segments.entries);
  return a.D == 128 ? launch<128>(a, maps, (int)grid, st) : launch<64>(a, maps, (int)grid, st);
}

__global__ void __launch_bounds__(1024) la_order_kernel(const int* bounds, int n_seqs, int* order) {
  after_previous();
  __shared__ int s_at[256];  // classes from the longest on: how many, then where the next one goes
  const int tid = threadIdx.x;
  auto cls = [&](int n) { return 255 - min((bounds[n + 1] - bounds[n] + kChunk - 1) / kChunk, 255); };
  if (tid < 256) s_at[tid] = 0;
  __syncthreads();
  for (int n = tid; n < n_seqs; n += 1024) atomicAdd(&s_at[cls(n)], 1);
  __syncthreads();
  if (tid < 32) {
    int v[8], sum = 0;
    for (int i = 0; i < 8; ++i) {
      v[i] = sum;
      sum += s_at[8 * tid + i];
    }
    int before = sum;
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, before, o);
      if (tid >= o) before += y;
    }
    for (int i = 0; i < 8; ++i) s_at[8 * tid + i] = before - sum + v[i];
  }
  __syncthreads();
  for (int n = tid; n < n_seqs; n += 1024) order[atomicAdd(&s_at[cls(n)], 1)] = n;
}
int launch_order(const int* bounds, int n_seqs, int* order, cudaStream_t st) {
  begin_stage(kStageOffsets, st);
  const int rc = launch_kernel(la_order_kernel, 1, 1024, 0, st, bounds, n_seqs, order);
  end_stage(st);
  return rc;
}

// Four elements a thread.  The entries do not wait for one another: eight at a time are asked for before the first is changed.
__global__ void __launch_bounds__(128) la_combine_kernel(const Call c, const Segments sg, int DD, int reverse, const float* init, float* states,
                                                         const double* decay) {
  after_previous();
  const int H = c.geo.heads, n = blockIdx.x / H, h = blockIdx.x - n * H, at = 4 * (blockIdx.y * 128 + threadIdx.x);
  const SeqInfo sq = gdr::sequence(c.geo, n);
  const int last = (sq.nchunks + sg.chunks - 1) / sg.chunks - 1;
  const size_t entry0 = (size_t)first_entry(c.geo, sg, n) * H + h;
  float4 R = init ? *reinterpret_cast<const float4*>(init + (size_t)blockIdx.x * DD + at) : make_float4(0.f, 0.f, 0.f, 0.f);
  for (int i0 = 0; i0 < last; i0 += 8) {
    float4 x[8];
    const auto index = [&](int k) { return entry0 + (size_t)(reverse ? last - i0 - k : i0 + k) * H; };
    // A lane has the decay of one of them.  Chunk by chunk a state may pass through one that no number holds: what leads out of this
    // range goes to R first, as a power of two (exact, or out of R's range as the result is) in two steps.
    const int mine = threadIdx.x & 7;
    const double d = i0 + mine < last ? decay[index(mine)] : 0.0;
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (i0 + k < last) x[k] = *reinterpret_cast<const float4*>(states + index(k) * DD + at);
    const long long fixed = __double2ll_rn(fmax(d, -4096.0) * (double)(1ll << kFixed));
    const int w = (int)(fixed >> kFixed), out = min(max(w - min(max(w, -60), 100), -252), 252);
    const float2 a = exp2_fixed_two(fixed - ((long long)out << kFixed));
    const bool far = __any_sync(0xffffffffu, out);
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const float2 by = f2(__shfl_sync(0xffffffffu, a.x, k), __shfl_sync(0xffffffffu, a.y, k));
      if (far) {
        const int up = __shfl_sync(0xffffffffu, out, k);
        const float p0 = __int_as_float((up / 2 + 127) << 23), p1 = __int_as_float((up - up / 2 + 127) << 23);
        R = make_float4(R.x * p0 * p1, R.y * p0 * p1, R.z * p0 * p1, R.w * p0 * p1);
      }
      if (i0 + k < last) {
        R.x = fmaf(R.x, by.x, fmaf(R.x, by.y, x[k].x));
        R.y = fmaf(R.y, by.x, fmaf(R.y, by.y, x[k].y));
        R.z = fmaf(R.z, by.x, fmaf(R.z, by.y, x[k].z));
        R.w = fmaf(R.w, by.x, fmaf(R.w, by.y, x[k].w));
        *reinterpret_cast<float4*>(states + index(k) * DD + at) = R;
      }
    }
  }
}

int combine_states(const Call& c, const Segments& s, int D, int reverse, const float* init, float* states, const double* decay, cudaStream_t st) {
  begin_stage(kStageLaStates, st);
  const int rc = launch_kernel(la_combine_kernel, dim3(c.geo.n_seqs * c.geo.heads, D * D / 512), 128, 0, st, c, s, D * D, reverse, init, states,
                               decay);
  end_stage(st);
  return rc;
}

}  // namespace la
}  // namespace pkda
