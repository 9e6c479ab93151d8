// Entry points of the gated delta rule: checks, scratch, and which kernels a call takes.
//
// bf16 activations of 128-channel heads take the chunked tensor-core kernels, everything else the token-by-token ones.
#include "gdr_common.cuh"
#include "gdr_tc.cuh"

namespace pkda {
namespace gdr {

static int check(const pkda_gdr_problem& p) {
  if (p.n_seqs < 0 || p.total_tokens < 0 || p.key_heads <= 0 || p.value_heads <= 0 || p.value_heads % p.key_heads) return PKDA_ERR_SHAPE;
  const int D = p.head_dim;
  if (D != 8 && D != 16 && D != 32 && D != 64 && D != 128) return PKDA_ERR_SHAPE;
  if (!p.cu_seqlens && (p.seq_len < 0 || (long long)p.n_seqs * p.seq_len != p.total_tokens)) return PKDA_ERR_SHAPE;
  // grids: four CTAs a (sequence, head), key heads as the second axis
  if ((long long)p.n_seqs * p.value_heads > (1ll << 28) || p.value_heads > 65535) return PKDA_ERR_SHAPE;
  if (p.dtype != PKDA_BF16 && p.dtype != PKDA_F32 && p.dtype != (PKDA_BF16 | PKDA_GDR_BETA_F32)) return PKDA_ERR_DTYPE;
  if (p.n_seqs == 0 || p.total_tokens == 0) return PKDA_OK;
  if (!p.q || !p.k || !p.v || !p.g || !p.beta) return PKDA_ERR_NULL;
  if (!aligned({p.q, p.k, p.v, p.initial_state}, 16)) return PKDA_ERR_ALIGN;
  return PKDA_OK;
}

static Params params(const pkda_gdr_problem& p, const int* bounds, const int* chunk_offsets) {
  Params b;
  b.geo.n_seqs = p.n_seqs;
  b.geo.seq_len = p.cu_seqlens ? 0 : p.seq_len;
  b.geo.total_tokens = p.total_tokens;
  b.geo.heads = p.value_heads;
  b.geo.chunks_per_seq = p.cu_seqlens ? 0 : (p.seq_len + kChunk - 1) / kChunk;
  b.geo.total_chunks = (int)chunk_count(p);
  b.geo.cu_seqlens = p.cu_seqlens ? (bounds ? bounds : p.cu_seqlens) : nullptr;
  b.geo.chunk_offsets = p.cu_seqlens ? chunk_offsets : nullptr;
  b.key_heads = p.key_heads;
  b.group = p.value_heads / p.key_heads;
  b.scale = p.scale;
  b.q = p.q; b.k = p.k; b.v = p.v; b.g = p.g; b.beta = p.beta; b.beta32 = beta_in_fp32(p); b.S0 = p.initial_state;
  return b;
}

// Packed batches: the sequences' bounds, never decreasing and inside the tensors whatever the caller's offsets hold, and
// the first chunk of each.  One CTA, 1,024 sequences a turn.
__global__ void __launch_bounds__(1024) gdr_offsets_kernel(const int* cu, int n_seqs, int total, int* bounds, int* offs) {
  after_previous();
  __shared__ int s_max[32], s_sum[32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  int before_max = min(max(cu[0], 0), total), before_sum = 0;
  if (tid == 0) {
    bounds[0] = before_max;
    offs[0] = 0;
  }
  for (int n0 = 0; n0 < n_seqs; n0 += 1024) {
    const int n = n0 + tid;
    int end = n < n_seqs ? min(max(cu[n + 1], 0), total) : 0;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, end, o);
      if (lane >= o) end = max(end, y);
    }
    if (lane == 31) s_max[warp] = end;
    __syncthreads();
    int start = before_max, all = before_max;
    for (int w = 0; w < 32; ++w) {
      if (w < warp) start = max(start, s_max[w]);
      all = max(all, s_max[w]);
    }
    end = max(end, start);
    int bos = __shfl_up_sync(0xffffffffu, end, 1);
    if (lane == 0) bos = start;
    int x = n < n_seqs ? (end - bos + kChunk - 1) / kChunk : 0;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += y;
    }
    if (lane == 31) s_sum[warp] = x;
    __syncthreads();
    int first = before_sum, sum = before_sum;
    for (int w = 0; w < 32; ++w) {
      if (w < warp) first += s_sum[w];
      sum += s_sum[w];
    }
    if (n < n_seqs) {
      bounds[n + 1] = end;
      offs[n + 1] = first + x;
    }
    before_max = all;
    before_sum = sum;
    __syncthreads();
  }
}

// Rows of a packed batch that no sequence owns (in front of the first, behind the last) get zeros.
__global__ void __launch_bounds__(256) gdr_unowned_rows_kernel(const int* cu, int n_seqs, int total, Rows r) {
  after_previous();
  int first = min(max(cu[0], 0), total), end = first;
  for (int n = 1 + threadIdx.x % 32; n <= n_seqs; n += 32) end = max(end, min(cu[n], total));
#pragma unroll
  for (int o = 16; o; o >>= 1) end = max(end, __shfl_xor_sync(0xffffffffu, end, o));
  for (int i = 0; i < 5; ++i) {
    if (!r.ptr[i]) continue;
    unsigned short* base = static_cast<unsigned short*>(r.ptr[i]);
    const long long row = r.bytes[i] / 2, at0 = blockIdx.x * 256ll + threadIdx.x, step = gridDim.x * 256ll;
    for (long long at = at0; at < first * row; at += step) base[at] = 0;
    for (long long at = end * row + at0; at < total * row; at += step) base[at] = 0;
  }
}

int launch_unowned_rows(const int* cu, int n_seqs, int total, const Rows& r, cudaStream_t st) {
  begin_stage(kStageGdrRows, st);
  const int rc = launch_kernel(gdr_unowned_rows_kernel, 64, 256, 0, st, cu, n_seqs, total, r);
  end_stage(st);
  return rc;
}
static int zero_unowned(const pkda_gdr_problem& p, const Rows& r, cudaStream_t st) {
  return p.cu_seqlens ? launch_unowned_rows(p.cu_seqlens, p.n_seqs, p.total_tokens, r, st) : PKDA_OK;
}

static long long act_bytes(const pkda_gdr_problem& p) { return act_dtype(p) == PKDA_BF16 ? 2 : 4; }

// No tokens: the states go through as they are.
static int empty_call(const pkda_gdr_problem& p, float* out, const float* in, cudaStream_t st) {
  if (!out || p.n_seqs == 0) return PKDA_OK;
  const size_t bytes = (size_t)p.n_seqs * p.value_heads * p.head_dim * p.head_dim * 4;
  if (in == out) return PKDA_OK;
  const cudaError_t err = in ? cudaMemcpyAsync(out, in, bytes, cudaMemcpyDeviceToDevice, st) : cudaMemsetAsync(out, 0, bytes, st);
  return launch_code(err);
}

int recurrent_forward(const pkda_gdr_recurrent_args* a, cudaStream_t st) {
  const pkda_gdr_problem& p = a->p;
  int rc = check(p);
  if (rc != PKDA_OK) return rc;
  if (!aligned({a->final_state}, 16)) return PKDA_ERR_ALIGN;
  if (p.total_tokens == 0) return empty_call(p, a->final_state, p.initial_state, st);
  if (!a->o) return PKDA_ERR_NULL;
  if (!aligned({a->o}, 16)) return PKDA_ERR_ALIGN;
  if (p.n_seqs) rc = exact_forward(p, params(p, nullptr, nullptr), a->o, a->final_state, nullptr, nullptr, st);
  if (rc != PKDA_OK) return rc;
  Rows r = {};
  r.ptr[0] = a->o;
  r.bytes[0] = p.value_heads * (long long)p.head_dim * act_bytes(p);
  return zero_unowned(p, r, st);
}

// ---- scratch and saved buffers, carved in the order below
struct Carver {
  char* base;
  size_t used = 0;
  template <typename X> X* take(size_t count) {
    X* at = reinterpret_cast<X*>(base + used);
    used = align_up(used + count * sizeof(X));
    return at;
  }
};

static bool chunked(const pkda_gdr_problem& p) { return act_dtype(p) == PKDA_BF16 && p.head_dim == kW; }

// A scan of few (row, head) units leaves most SMs idle, and the kernel in front of the forward's (the pairs) or behind the
// reverse one (the gradients) works on chunks one by one.  So a dense call is taken in two parts: the scan of the first
// chunks runs beside the pairs of the others, the reverse scan of the first chunks beside the gradients of the others.  What is computed
// stays the same, bit for bit.  Returns the chunks of a sequence that come first, 0 to take all at once.
//
// A scan takes 2.8 us a chunk (reverse 4.1), whatever the units; the other kernel 24 ns (55) a chunk and unit with all SMs.  Beside the
// scan it has those that the units leave; both are to take as long.  Single calls at once / in two parts: forward of 8,191 tokens of
// 16 heads 420 / 391 us, of 2 x 4,096 249 / 220, forward and backward 1,214 / 1,119 and 722 / 647; 64 units (4 x 4,096) 883 / 802.
// The pairs' latency does not shrink with their number: forwards of short rows or less than two of their CTAs an SM gain
// nothing (1,100 tokens of 64 heads 88 / 96 us, 2 x 2,047 of 4 key heads 121 / 125) and are taken at once.
constexpr int kPartChunks = 16;
static size_t between_parts(const pkda_gdr_problem& p) {  // floats of the states that pass from part to part
  const size_t units = (size_t)p.n_seqs * p.value_heads;
  return !p.cu_seqlens && p.seq_len > kPartChunks * kChunk && units <= 128 ? units * p.head_dim * p.head_dim : 0;
}
static int first_part(const pkda_gdr_problem& p, bool reverse) {
  const long long units = (long long)p.n_seqs * p.value_heads, sms = sm_count();
  if (!between_parts(p) || 2 * units > sms) return 0;
  const long long chunks = (p.seq_len + kChunk - 1) / kChunk;
  if (!reverse && (chunks < 2 * kPartChunks || chunks * p.n_seqs * p.key_heads < 2 * sms)) return 0;
  const long long other = (reverse ? 6 : 4) * units, scan = 3 * (sms - units);
  return (int)((chunks * other + other + scan - 1) / (other + scan));
}

struct Saved {  // left by a forward for its backward
  int *bounds, *offs;  // packed batches
  float *e, *h;        // token-by-token kernels
  ChunkBuffers c;      // chunked kernels
  float* between;      // (scratch) states between two parts
};
static size_t carve_saved(const pkda_gdr_problem& p, void* base, Saved* s) {
  Carver c{static_cast<char*>(base)};
  const size_t rows = (size_t)p.total_tokens * p.value_heads, items = chunk_count(p) * p.value_heads, D = p.head_dim;
  s->bounds = c.take<int>((size_t)p.n_seqs + 1);
  s->offs = c.take<int>((size_t)p.n_seqs + 1);
  if (chunked(p)) {
    s->c.T2 = c.take<bf16>(items * 2 * 64 * 64);
    s->c.P = c.take<bf16>(items * 2 * 64 * 64);
    s->c.scal = c.take<float>(items * kScalars);
    s->c.e = c.take<bf16>(items * 2 * D * 64);
    s->c.h = c.take<bf16>(items * 2 * D * D);
  } else {
    s->e = c.take<float>(rows * D);
    s->h = c.take<float>(items * D * D);
  }
  return c.used;
}
size_t saved_bytes(const pkda_gdr_problem& p) {
  Saved s;
  return check(p) == PKDA_ERR_SHAPE ? 0 : carve_saved(p, nullptr, &s);
}

// The chunked forward's own scratch; where nothing is saved, what would be saved of it too.
static size_t carve_forward(const pkda_gdr_problem& p, void* base, bool save, Saved* s) {
  Carver c{static_cast<char*>(base)};
  const size_t items = chunk_count(p) * p.value_heads;
  s->c.status = c.take<int>(1);
  s->between = c.take<float>(between_parts(p));
  s->c.T = c.take<bf16>(items * 2 * 64 * 64);
  if (!save) {
    s->bounds = c.take<int>((size_t)p.n_seqs + 1);
    s->offs = c.take<int>((size_t)p.n_seqs + 1);
    s->c.P = c.take<bf16>(items * 2 * 64 * 64);
    s->c.scal = c.take<float>(items * kScalars);
    s->c.T2 = s->c.e = s->c.h = nullptr;
  }
  return c.used;
}
size_t fwd_workspace(const pkda_gdr_problem& p) {
  Saved s;
  return check(p) == PKDA_ERR_SHAPE || !chunked(p) ? 0 : carve_forward(p, nullptr, false, &s);
}

struct BwdScratch {
  float *y, *dh;  // token-by-token kernels
  GradBuffers g;  // chunked kernels
  float* between;
  int* status;
};
static size_t carve_backward(const pkda_gdr_problem& p, void* base, BwdScratch* s) {
  Carver c{static_cast<char*>(base)};
  const size_t items = chunk_count(p) * p.value_heads, D = p.head_dim;
  if (chunked(p)) {
    s->status = c.take<int>(1);
    s->between = c.take<float>(between_parts(p));
    s->g.y = c.take<bf16>(items * 2 * D * 64);
    s->g.dh = c.take<bf16>(items * 2 * D * D);
  } else {
    s->y = c.take<float>((size_t)p.total_tokens * p.value_heads * D);
    s->dh = c.take<float>(items * D * D);
  }
  return c.used;
}
size_t bwd_workspace(const pkda_gdr_problem& p) {
  BwdScratch s;
  return check(p) == PKDA_ERR_SHAPE ? 0 : carve_backward(p, nullptr, &s);
}

int launch_offsets(const int* cu, int n_seqs, int total, int* bounds, int* offs, cudaStream_t st) {
  begin_stage(kStageOffsets, st);
  const int rc = launch_kernel(gdr_offsets_kernel, 1, 1024, 0, st, cu, n_seqs, total, bounds, offs);
  end_stage(st);
  return rc;
}
static int order_offsets(const pkda_gdr_problem& p, int* bounds, int* offs, cudaStream_t st) {
  return p.cu_seqlens ? launch_offsets(p.cu_seqlens, p.n_seqs, p.total_tokens, bounds, offs, st) : PKDA_OK;
}

// (The testing aid of pkda_set_variant leaves it set, as a wait that gave up would.)
static int clear_status(int* status, cudaStream_t st) {
  const cudaError_t err = cudaMemsetAsync(status, stage_variant(kStageGdrScan), sizeof(int), st);
  return err == cudaSuccess ? PKDA_OK : launch_code(err);
}

static int chunk_forward(const pkda_gdr_fwd_args* a, Saved& s, cudaStream_t st) {
  const pkda_gdr_problem& p = a->p;
  if (!a->workspace || a->workspace_bytes < fwd_workspace(p)) return PKDA_ERR_WORKSPACE;
  carve_forward(p, a->workspace, a->saved != nullptr, &s);
  if (int err = clear_status(s.c.status, st)) return err;
  int rc = order_offsets(p, s.bounds, s.offs, st);
  if (rc != PKDA_OK) return rc;
  const Params b = params(p, s.bounds, s.offs);
  bf16* o = static_cast<bf16*>(a->o);
  Part first, rest;
  first.c1 = rest.c0 = first_part(p, false);
  rc = launch_pairs(b, s.c, first, st);
  if (rc != PKDA_OK) return rc;
  if (!first.c1) return launch_scan(b, s.c, first, p.initial_state, o, a->final_state, st);
  rest.c1 = b.geo.chunks_per_seq;
  first.ordinary = true;  // (the pairs beside it read the inputs and the offsets)
  rc = launch_scan(b, s.c, first, p.initial_state, o, s.between, st);
  rest.beside = true;
  if (rc == PKDA_OK) rc = launch_pairs(b, s.c, rest, st);
  rest.beside = false;
  return rc != PKDA_OK ? rc : launch_scan(b, s.c, rest, s.between, o, a->final_state, st);
}

int forward(const pkda_gdr_fwd_args* a, cudaStream_t st) {
  const pkda_gdr_problem& p = a->p;
  int rc = check(p);
  if (rc != PKDA_OK) return rc;
  if (!aligned({a->final_state, a->saved, a->workspace}, 16)) return PKDA_ERR_ALIGN;
  if (p.total_tokens == 0) return empty_call(p, a->final_state, p.initial_state, st);
  if (!a->o) return PKDA_ERR_NULL;
  if (!aligned({a->o}, 16)) return PKDA_ERR_ALIGN;
  Saved s = {};
  if (a->saved) {
    if (a->saved_bytes < saved_bytes(p)) return PKDA_ERR_WORKSPACE;
    carve_saved(p, a->saved, &s);
  }
  if (p.n_seqs == 0) {
    rc = PKDA_OK;  // (no row is anybody's)
  } else if (chunked(p)) {
    rc = chunk_forward(a, s, st);
  } else {
    if (a->saved) rc = order_offsets(p, s.bounds, s.offs, st);
    if (rc != PKDA_OK) return rc;
    rc = exact_forward(p, a->saved ? params(p, s.bounds, s.offs) : params(p, nullptr, nullptr), a->o, a->final_state, s.e, s.h, st);
  }
  if (rc != PKDA_OK) return rc;
  Rows r = {};
  r.ptr[0] = a->o;
  r.bytes[0] = p.value_heads * (long long)p.head_dim * act_bytes(p);
  return zero_unowned(p, r, st);
}

int backward(const pkda_gdr_bwd_args* a, cudaStream_t st) {
  const pkda_gdr_problem& p = a->p;
  int rc = check(p);
  if (rc != PKDA_OK) return rc;
  if (!aligned({a->d_o, a->d_final_state, a->saved, a->dq, a->dk, a->dv, a->d_initial_state, a->workspace}, 16)) return PKDA_ERR_ALIGN;
  if (p.total_tokens == 0) return empty_call(p, a->d_initial_state, a->d_final_state, st);
  if (!a->d_o || !a->saved || !a->dq || !a->dk || !a->dv || !a->dg || !a->dbeta) return PKDA_ERR_NULL;
  if (a->saved_bytes < saved_bytes(p) || !a->workspace || a->workspace_bytes < bwd_workspace(p)) return PKDA_ERR_WORKSPACE;
  Saved s;
  carve_saved(p, const_cast<void*>(a->saved), &s);
  BwdScratch w;
  carve_backward(p, a->workspace, &w);
  const Params b = params(p, s.bounds, s.offs);
  if (p.n_seqs == 0) {
    rc = PKDA_OK;
  } else if (chunked(p)) {
    s.c.status = w.status;
    if (int err = clear_status(w.status, st)) return err;
    const bf16* d_o = static_cast<const bf16*>(a->d_o);
    auto scan = [&](const Part& t, const float* from, float* to) {
      return launch_scan_bwd(b, s.c, w.g, t, d_o, from, static_cast<bf16*>(a->dv), to, st);
    };
    auto gradients = [&](const Part& t) {
      return launch_grad(b, s.c, w.g, t, d_o, static_cast<bf16*>(a->dq), static_cast<bf16*>(a->dk), a->dg, a->dbeta, st);
    };
    Part first, rest;
    first.c1 = rest.c0 = first_part(p, true);
    if (first.c1) {
      rest.c1 = b.geo.chunks_per_seq;
      rc = scan(rest, a->d_final_state, w.between);
      first.ordinary = true;  // (the gradients beside it read what the scan of the rest and the forward have left)
      if (rc == PKDA_OK) rc = scan(first, w.between, a->d_initial_state);
      rest.beside = true;
      if (rc == PKDA_OK) rc = gradients(rest);
    } else {
      rc = scan(first, a->d_final_state, a->d_initial_state);
    }
    if (rc == PKDA_OK) rc = gradients(first);
  } else {
    rc = exact_backward(p, b, *a, s.e, s.h, w.y, w.dh, st);
  }
  if (rc != PKDA_OK) return rc;
  Rows r = {};
  const long long act = act_bytes(p), D = p.head_dim;
  r.ptr[0] = a->dq; r.bytes[0] = p.key_heads * D * act;
  r.ptr[1] = a->dk; r.bytes[1] = p.key_heads * D * act;
  r.ptr[2] = a->dv; r.bytes[2] = p.value_heads * D * act;
  r.ptr[3] = a->dg; r.bytes[3] = p.value_heads * 4;
  r.ptr[4] = a->dbeta; r.bytes[4] = p.value_heads * (beta_in_fp32(p) ? 4 : 2);
  return zero_unowned(p, r, st);
}

}  // namespace gdr
}  // namespace pkda

extern "C" {

int pkda_gdr_recurrent_fwd(const pkda_gdr_recurrent_args* args, void* cuda_stream) {
  if (!args) return PKDA_ERR_NULL;
  pkda::reset_launch_count();
  return pkda::gdr::recurrent_forward(args, static_cast<cudaStream_t>(cuda_stream));
}
size_t pkda_gdr_saved_bytes(const pkda_gdr_problem* p) { return p ? pkda::gdr::saved_bytes(*p) : 0; }
size_t pkda_gdr_fwd_workspace_bytes(const pkda_gdr_problem* p) { return p ? pkda::gdr::fwd_workspace(*p) : 0; }
int pkda_gdr_fwd(const pkda_gdr_fwd_args* args, void* cuda_stream) {
  if (!args) return PKDA_ERR_NULL;
  pkda::reset_launch_count();
  return pkda::gdr::forward(args, static_cast<cudaStream_t>(cuda_stream));
}
size_t pkda_gdr_bwd_workspace_bytes(const pkda_gdr_problem* p) { return p ? pkda::gdr::bwd_workspace(*p) : 0; }
int pkda_gdr_bwd(const pkda_gdr_bwd_args* args, void* cuda_stream) {
  if (!args) return PKDA_ERR_NULL;
  pkda::reset_launch_count();
  return pkda::gdr::backward(args, static_cast<cudaStream_t>(cuda_stream));
}
size_t pkda_sizeof_gdr_problem(void) { return sizeof(pkda_gdr_problem); }
size_t pkda_sizeof_gdr_recurrent_args(void) { return sizeof(pkda_gdr_recurrent_args); }
size_t pkda_sizeof_gdr_fwd_args(void) { return sizeof(pkda_gdr_fwd_args); }
size_t pkda_sizeof_gdr_bwd_args(void) { return sizeof(pkda_gdr_bwd_args); }

}  // extern "C"
