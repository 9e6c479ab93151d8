// Entry points of linear attention: checks, scratch, and which kernels a call takes.
//
// bf16 activations of heads of 128 and 64 channels take the chunked tensor-core kernels, everything else the token-by-token ones.
#include "la_common.cuh"
#include "la_tc.cuh"

#include <cmath>

namespace pkda {
namespace la {

static int check(const pkda_la_problem& p) {
  if (p.n_seqs < 0 || p.total_tokens < 0 || p.key_heads <= 0 || p.value_heads <= 0 || p.value_heads % p.key_heads) return PKDA_ERR_SHAPE;
  const int D = p.head_dim;
  if (D != 8 && D != 16 && D != 32 && D != 64 && D != 128) return PKDA_ERR_SHAPE;
  if (!p.cu_seqlens && (p.seq_len < 0 || (long long)p.n_seqs * p.seq_len != p.total_tokens)) return PKDA_ERR_SHAPE;
  // grids: eight CTAs a (sequence, head), or one for each segment of it
  if (((long long)p.n_seqs + p.total_tokens / kChunk) * p.value_heads > (1ll << 27)) return PKDA_ERR_SHAPE;
  if (p.dtype != PKDA_BF16 && p.dtype != PKDA_F32) return PKDA_ERR_DTYPE;
  if (p.n_seqs == 0 || p.total_tokens == 0) return PKDA_OK;
  if (!p.q || !p.k || !p.v || !p.g) return PKDA_ERR_NULL;
  if (!aligned({p.q, p.k, p.v, p.initial_state}, 16) || !aligned({p.g, p.cu_seqlens}, 4)) return PKDA_ERR_ALIGN;
  return PKDA_OK;
}

static Call call(const pkda_la_problem& p, const int* bounds, const int* offs) {
  Call c;
  c.geo.n_seqs = p.n_seqs;
  c.geo.seq_len = p.cu_seqlens ? 0 : p.seq_len;
  c.geo.total_tokens = p.total_tokens;
  c.geo.heads = p.value_heads;
  c.geo.chunks_per_seq = p.cu_seqlens ? 0 : (p.seq_len + kChunk - 1) / kChunk;
  c.geo.total_chunks = 0;
  c.geo.cu_seqlens = p.cu_seqlens ? (bounds ? bounds : p.cu_seqlens) : nullptr;
  c.geo.chunk_offsets = p.cu_seqlens ? offs : nullptr;
  c.g = p.g;
  c.g_step = p.gate_per_head ? 0 : p.value_heads;
  return c;
}

static long long act_bytes(const pkda_la_problem& p) { return p.dtype == PKDA_BF16 ? 2 : 4; }
static size_t units(const pkda_la_problem& p) { return (size_t)p.n_seqs * p.value_heads; }
static size_t states(const pkda_la_problem& p) { return units(p) * p.head_dim * p.head_dim; }

// No tokens: the states go through as they are.
static int empty_call(const pkda_la_problem& p, float* out, const float* in, cudaStream_t st) {
  if (!out || p.n_seqs == 0 || in == out) return PKDA_OK;
  const size_t bytes = states(p) * sizeof(float);
  const cudaError_t err = in ? cudaMemcpyAsync(out, in, bytes, cudaMemcpyDeviceToDevice, st) : cudaMemsetAsync(out, 0, bytes, st);
  return launch_code(err);
}

static Pass forward_pass(const pkda_la_problem& p, void* o, float* final_state) {
  Pass f = {};
  const int group = p.value_heads / p.key_heads;
  f.x = p.q; f.y = p.k; f.z = p.v;
  f.x_group = f.y_group = group; f.z_group = f.u_group = 1;
  f.init = p.initial_state; f.fin = final_state;
  f.out = o;
  f.c = f.read = p.scale; f.write = 1.f;
  return f;
}

static int zero_unowned(const pkda_la_problem& p, const gdr::Rows& r, cudaStream_t st) {
  return p.cu_seqlens ? gdr::launch_unowned_rows(p.cu_seqlens, p.n_seqs, p.total_tokens, r, st) : PKDA_OK;
}
static int zero_unowned(const pkda_la_problem& p, void* o, cudaStream_t st) {
  gdr::Rows r = {};
  r.ptr[0] = o;
  r.bytes[0] = p.value_heads * (long long)p.head_dim * act_bytes(p);
  return zero_unowned(p, r, st);
}

int recurrent_forward(const pkda_la_recurrent_args* a, cudaStream_t st) {
  const pkda_la_problem& p = a->p;
  int rc = check(p);
  if (rc != PKDA_OK) return rc;
  if (!aligned({a->final_state}, 16)) return PKDA_ERR_ALIGN;
  if (p.total_tokens == 0) return empty_call(p, a->final_state, p.initial_state, st);
  if (!a->o) return PKDA_ERR_NULL;
  if (!aligned({a->o}, 16)) return PKDA_ERR_ALIGN;
  if (p.n_seqs) {
    const Pass f = forward_pass(p, a->o, a->final_state);
    const Call c = call(p, nullptr, nullptr);
    rc = takes_step(c, p.head_dim) ? launch_step(c, p.head_dim, p.dtype, f, st) : launch_chain(c, p.head_dim, p.dtype, &f, 1, ChainEnds(), st);
  }
  return rc != PKDA_OK ? rc : zero_unowned(p, a->o, st);
}

// ---- how a call is cut, scratch and saved buffers
// Which calls the chunked kernels take.
static bool chunked(const pkda_la_problem& p) { return p.dtype == PKDA_BF16 && (p.head_dim == 128 || p.head_dim == 64); }

// Segments.  The forward leaves a state for the backward at each end (64 KB for the 1 MB that a head of 128 channels has
// read and written by then, at sixteen chunks a segment), and the gate's gradient starts anew from <S, dS> there.  Shorter ones where that gives more SMs a part of the call.
constexpr int kMostChunks = 16, kLeastChunks = 4;
static int chunks_of(const pkda_la_problem& p) {  // of a sequence; packed: in the mean
  if (p.cu_seqlens) return (int)(((long long)p.total_tokens / kChunk + p.n_seqs) / (p.n_seqs > 0 ? p.n_seqs : 1));
  return (p.seq_len + kChunk - 1) / kChunk;
}
static Segments segments(const pkda_la_problem& p) {
  Segments s;
  const int chunks = chunks_of(p), side = (int)(sm_count() / (units(p) ? units(p) : 1));  // segments of each sequence that SMs have room for
  s.chunks = side > 1 ? (chunks + side - 1) / side : kMostChunks;
  s.chunks = s.chunks < kLeastChunks || !chunked(p) ? kLeastChunks : s.chunks > kMostChunks ? kMostChunks : s.chunks;
  if (p.cu_seqlens) {
    s.entries = ((long long)p.total_tokens / kChunk + p.n_seqs) / s.chunks + p.n_seqs;
  } else {
    s.segs = chunks > s.chunks ? (chunks + s.chunks - 1) / s.chunks : 1;
    s.entries = (long long)p.n_seqs * s.segs;
  }
  return s;
}
// Whether the segments of a sequence run side by side, from states that a pass over the keys and values (or queries and cotangents) has left, or one
// CTA walks from one to the next.  In chunks of a walk, `n` of them side by side (two and the segments of dq, backwards): the pass over states alone takes 0.5
// of one, and it and what puts its states together cost 4 more.  Forward of 8,191 tokens of 16 heads: 220 us walked, 80
// side by side.
static bool side_by_side(const pkda_la_problem& p, int n) {
  const Segments s = segments(p);
  const double sms = sm_count(), u = (double)units(p), chunks = chunks_of(p), segs = ceil(chunks / s.chunks);
  const double walk = fmax(chunks, n * u * chunks / sms), all = ceil(n * u * segs / sms) * s.chunks;
  return segs > 1 && 0.5 * ceil(u * (segs - 1) / sms) * s.chunks + all + 4 < walk;
}
// Whether walks of a packed batch take its sequences by their length: where not all of them start at once.  (22 documents of 170 to 3,899
// tokens, 16 heads: forward 170 us, 203 in their own order; backward 860 either way, its three operations follow one another anyway.)
static bool ordered(const pkda_la_problem& p) { return p.cu_seqlens && chunked(p) && p.n_seqs > 1 && 3 * (long long)units(p) > sm_count(); }
static size_t segment_states(const pkda_la_problem& p) { return (size_t)segments(p).entries * p.value_heads * p.head_dim * p.head_dim; }

struct Carver {
  char* base;
  size_t used = 0;
  template <typename X> X* take(size_t count) {
    X* at = reinterpret_cast<X*>(base + used);
    used = align_up(used + count * sizeof(X));
    return at;
  }
};

struct Saved {  // left by a forward for its backward
  int *bounds, *offs;  // packed batches
  int* order;          // and the order of their walks
  float* S;            // states at the segments' ends
};
static size_t carve_saved(const pkda_la_problem& p, void* base, Saved* s) {
  Carver c{static_cast<char*>(base)};
  s->bounds = c.take<int>((size_t)p.n_seqs + 1);
  s->offs = c.take<int>((size_t)p.n_seqs + 1);
  s->order = c.take<int>(ordered(p) ? p.n_seqs : 0);
  s->S = c.take<float>(segment_states(p));
  return c.used;
}
size_t saved_bytes(const pkda_la_problem& p) {
  Saved s;
  return check(p) == PKDA_ERR_SHAPE ? 0 : carve_saved(p, nullptr, &s);
}

// The chunked forward's own scratch; where nothing is saved, what would be saved of it too.
struct FwdScratch {
  int *status, *bounds, *offs, *order;
  float* S;       // segments side by side: their states
  double* decay;  // and decays
};
static size_t carve_forward(const pkda_la_problem& p, void* base, FwdScratch* s) {
  Carver c{static_cast<char*>(base)};
  s->status = c.take<int>(1);
  s->bounds = c.take<int>((size_t)p.n_seqs + 1);
  s->offs = c.take<int>((size_t)p.n_seqs + 1);
  s->order = c.take<int>(ordered(p) ? p.n_seqs : 0);
  const bool split = side_by_side(p, 1);  // (for a call in place too, which walks)
  s->S = c.take<float>(split ? segment_states(p) : 0);
  s->decay = c.take<double>(split ? (size_t)segments(p).entries * p.value_heads : 0);
  return c.used;
}
size_t fwd_workspace(const pkda_la_problem& p) {
  FwdScratch s;
  return check(p) == PKDA_ERR_SHAPE || !chunked(p) ? 0 : carve_forward(p, nullptr, &s);
}

struct BwdScratch {
  int* status;
  float *dq, *dk;    // of each value head, where they share key heads
  float *row, *col;  // the gate's gradient
  float* X;
  int* grows;
  double* part;
  float* R;          // segments side by side: the states' cotangents
  double* decay;     // and decays
};
static int row_slices(const pkda_la_problem& p) { return chunked(p) ? read_slices(p.head_dim) : chain_slices((long long)units(p), p.head_dim); }
static int x_parts(const pkda_la_problem& p) { return chunked(p) ? kXParts : chain_x_parts((long long)units(p), p.head_dim); }
static int col_slices(const pkda_la_problem& p) { return row_slices(p) + (chunked(p) ? kPairSlices : 0); }
static size_t carve_backward(const pkda_la_problem& p, void* base, BwdScratch* s) {
  Carver c{static_cast<char*>(base)};
  const size_t rows = (size_t)p.total_tokens * p.value_heads, entries = (size_t)segments(p).entries * p.value_heads;
  const bool shared = p.value_heads != p.key_heads;
  s->status = c.take<int>(1);
  s->dq = c.take<float>(shared ? rows * p.head_dim : 0);
  s->dk = c.take<float>(shared ? rows * p.head_dim : 0);
  s->row = c.take<float>(row_slices(p) * rows);
  s->col = c.take<float>(col_slices(p) * rows);
  s->X = c.take<float>(entries * x_parts(p));
  s->grows = c.take<int>(chunked(p) ? entries : 0);
  s->part = c.take<double>(p.gate_per_head ? entries : 0);
  const bool split = chunked(p) && side_by_side(p, 3);
  s->R = c.take<float>(split ? segment_states(p) : 0);
  s->decay = c.take<double>(split ? entries : 0);
  return c.used;
}
size_t bwd_workspace(const pkda_la_problem& p) {
  BwdScratch s;
  return check(p) == PKDA_ERR_SHAPE ? 0 : carve_backward(p, nullptr, &s);
}

// (The testing aid of pkda_set_variant leaves it set, as a wait that gave up would.)
static int clear_status(int* status, cudaStream_t st) {
  const cudaError_t err = cudaMemsetAsync(status, stage_variant(kStageLaChunks), sizeof(int), st);
  return err == cudaSuccess ? PKDA_OK : launch_code(err);
}

static ChunkCall chunk_call(const pkda_la_problem& p, const Call& c, int* status, const void* d_o) {
  ChunkCall a = {};
  a.c = c;
  a.segments = segments(p);
  a.D = p.head_dim;
  a.status = status;
  a.base[0] = p.q; a.base[1] = p.k; a.base[2] = p.v; a.base[3] = d_o;
  a.heads[0] = a.heads[1] = p.key_heads; a.heads[2] = a.heads[3] = p.value_heads;
  return a;
}
enum { kMapQ, kMapK, kMapV, kMapDo };
static ChunkPass chunk_pass(const Pass& p, int x, int y, int z, int u) {
  ChunkPass t = {};
  t.p = p;
  t.map[0] = x; t.map[1] = y; t.map[2] = z; t.map[3] = u;
  return t;
}

// The states between segments for an operation whose segments run side by side: `entry` k is R at its end in the direction of time.
static int states_between(const ChunkCall& of, const ChunkPass& pass, float* states, double* decay, cudaStream_t st) {
  ChunkCall a = of;
  a.n = 1;
  ChunkPass& t = a.pass[0];
  t = pass;
  t.p.out = t.p.fin = t.p.dots = nullptr;
  t.p.u = nullptr;
  t.walk = t.reads = t.pairs = 0;
  t.X = nullptr;
  t.states_only = 1;
  t.ends = states;
  t.decay = decay;
  if (int rc = launch_chunks(a, st)) return rc;
  return combine_states(a.c, a.segments, a.D, pass.p.reverse, pass.p.init, states, decay, st);
}

int forward(const pkda_la_fwd_args* a, cudaStream_t st) {
  const pkda_la_problem& p = a->p;
  int rc = check(p);
  if (rc != PKDA_OK) return rc;
  if (!aligned({a->final_state, a->saved, a->workspace}, 16)) return PKDA_ERR_ALIGN;
  if (p.total_tokens == 0) return empty_call(p, a->final_state, p.initial_state, st);
  if (!a->o) return PKDA_ERR_NULL;
  if (!aligned({a->o}, 16)) return PKDA_ERR_ALIGN;
  if (chunked(p) && (!a->workspace || a->workspace_bytes < fwd_workspace(p))) return PKDA_ERR_WORKSPACE;
  Saved s = {};
  if (a->saved) {
    if (a->saved_bytes < saved_bytes(p)) return PKDA_ERR_WORKSPACE;
    carve_saved(p, a->saved, &s);
  }
  if (p.n_seqs) {
    FwdScratch w = {};
    if (chunked(p)) {
      carve_forward(p, a->workspace, &w);
      if (!a->saved) {
        s.bounds = w.bounds;
        s.offs = w.offs;
        s.order = w.order;
      }
      if ((rc = clear_status(w.status, st)) != PKDA_OK) return rc;
    }
    if (s.bounds && p.cu_seqlens) rc = gdr::launch_offsets(p.cu_seqlens, p.n_seqs, p.total_tokens, s.bounds, s.offs, st);
    if (rc == PKDA_OK && ordered(p)) rc = launch_order(s.bounds, p.n_seqs, s.order, st);
    if (rc != PKDA_OK) return rc;
    const Call c = call(p, s.bounds, s.offs);
    Pass f = forward_pass(p, a->o, a->final_state);
    if (chunked(p)) {
      ChunkCall k = chunk_call(p, c, w.status, nullptr);
      k.n = 1;
      k.order = ordered(p) ? s.order : nullptr;
      k.pass[0] = chunk_pass(f, kMapQ, kMapK, kMapV, 0);
      k.pass[0].ends = s.S;
      const bool in_place = a->final_state && a->final_state == p.initial_state;  // (the first segment could find the last one's state)
      k.pass[0].walk = in_place || !side_by_side(p, 1);
      if (!k.pass[0].walk) {
        float* states = s.S ? s.S : w.S;
        k.pass[0].starts = states;
        rc = states_between(k, k.pass[0], states, w.decay, st);
      }
      if (rc == PKDA_OK) rc = launch_chunks(k, st);
    } else {
      ChainEnds ends;
      ends.segments = segments(p);
      ends.ends = s.S;
      rc = launch_chain(c, p.head_dim, p.dtype, &f, 1, ends, st);
    }
  }
  return rc != PKDA_OK ? rc : zero_unowned(p, a->o, st);
}

int backward(const pkda_la_bwd_args* a, cudaStream_t st) {
  const pkda_la_problem& p = a->p;
  int rc = check(p);
  if (rc != PKDA_OK) return rc;
  if (!aligned({a->d_o, a->d_final_state, a->saved, a->dq, a->dk, a->dv, a->d_initial_state, a->workspace}, 16) || !aligned({a->dg}, 4))
    return PKDA_ERR_ALIGN;
  if (p.total_tokens == 0) {
    if (p.gate_per_head && a->dg && cudaMemsetAsync(a->dg, 0, p.value_heads * sizeof(float), st) != cudaSuccess) return PKDA_ERR_LAUNCH;
    return empty_call(p, a->d_initial_state, a->d_final_state, st);
  }
  if (!a->d_o || !a->saved || !a->dq || !a->dk || !a->dv) return PKDA_ERR_NULL;
  if (a->saved_bytes < saved_bytes(p) || !a->workspace || a->workspace_bytes < bwd_workspace(p)) return PKDA_ERR_WORKSPACE;
  Saved s;
  carve_saved(p, const_cast<void*>(a->saved), &s);
  BwdScratch w;
  carve_backward(p, a->workspace, &w);
  const int group = p.value_heads / p.key_heads, D = p.head_dim;
  if (p.n_seqs) {
    const Call c = call(p, s.bounds, s.offs);
    Pass q = {}, k = {}, v = {};
    q.x = a->d_o; q.y = p.v; q.z = p.k; q.u = p.q;
    q.x_group = q.y_group = 1; q.z_group = q.u_group = group;
    q.init = p.initial_state; q.init_t = 1;
    q.c = q.read = p.scale; q.write = 1.f;
    k.x = p.v; k.y = a->d_o; k.z = p.q; k.u = p.k;
    k.x_group = k.y_group = 1; k.z_group = k.u_group = group;
    k.init = a->d_final_state; k.init_t = 1;
    k.c = k.write = p.scale; k.read = 1.f; k.reverse = 1;
    v.x = p.k; v.y = p.q; v.z = a->d_o;
    v.x_group = v.y_group = group; v.z_group = v.u_group = 1;
    v.init = a->d_final_state; v.fin = a->d_initial_state;
    v.c = v.write = p.scale; v.read = 1.f; v.reverse = 1;
    q.out = group > 1 ? w.dq : a->dq; q.out32 = group > 1;
    k.out = group > 1 ? w.dk : a->dk; k.out32 = group > 1;
    v.out = a->dv;
    if (a->dg) {
      q.dots = w.row;
      k.dots = w.col;
    } else {
      q.u = k.u = nullptr;
    }
    if (chunked(p)) {
      if ((rc = clear_status(w.status, st)) != PKDA_OK) return rc;
      ChunkCall t = chunk_call(p, c, w.status, a->d_o);
      t.n = 3;
      t.order = ordered(p) ? s.order : nullptr;
      ChunkPass &cv = t.pass[0], &ck = t.pass[1], &cq = t.pass[2];
      cv = chunk_pass(v, kMapK, kMapQ, kMapDo, 0);
      ck = chunk_pass(k, kMapV, kMapDo, kMapQ, kMapK);
      cq = chunk_pass(q, kMapDo, kMapV, kMapK, kMapQ);
      cv.walk = ck.walk = !side_by_side(p, 3);
      cv.starts = ck.starts = w.R;
      cq.starts = s.S;
      if (a->dg) {
        ck.reads = cq.reads = 1;
        ck.X_states = s.S;
        ck.X = w.X;
        ck.grows = w.grows;
        cv.pairs = 1;  // (k.q and v.do: on the operation that leaves no row sums)
        cv.map[3] = kMapV;
        cv.p.u = p.v;
        cv.p.dots = w.col + (size_t)row_slices(p) * p.total_tokens * p.value_heads;
      }
      if (!cv.walk) rc = states_between(t, cv, w.R, w.decay, st);
      if (rc == PKDA_OK) rc = launch_chunks(t, st);
    } else {
      const Pass t[3] = {q, k, v};
      ChainEnds ends;
      ends.segments = segments(p);
      if (a->dg) {
        ends.X_states = s.S;
        ends.X = w.X;
      }
      rc = launch_chain(c, D, p.dtype, t, 3, ends, st);
    }
    if (rc == PKDA_OK && a->dg) {
      GateGrad g = {};
      g.c = c;
      g.segments = segments(p);
      g.row = w.row; g.col = w.col;
      g.row_slices = row_slices(p); g.col_slices = col_slices(p);
      g.X = w.X; g.x_parts = x_parts(p);
      g.grows = chunked(p) ? w.grows : nullptr;
      g.S0 = p.initial_state; g.dS0 = a->d_initial_state;
      g.D = D;
      if (p.gate_per_head) {
        g.part = w.part;
        g.dg_head = a->dg;
      } else {
        g.dg = a->dg;
      }
      rc = launch_gate_grad(g, st);
    }
    if (rc == PKDA_OK && group > 1) rc = launch_group_sum(w.dq, a->dq, w.dk, a->dk, p.dtype, p.total_tokens, p.key_heads, group, D, st);
  } else if (p.gate_per_head && a->dg && cudaMemsetAsync(a->dg, 0, p.value_heads * sizeof(float), st) != cudaSuccess) {
    return PKDA_ERR_LAUNCH;
  }
  if (rc != PKDA_OK) return rc;
  gdr::Rows r = {};
  const long long act = act_bytes(p);
  r.ptr[0] = a->dq; r.bytes[0] = p.key_heads * D * act;
  r.ptr[1] = a->dk; r.bytes[1] = p.key_heads * D * act;
  r.ptr[2] = a->dv; r.bytes[2] = p.value_heads * D * act;
  r.ptr[3] = p.gate_per_head ? nullptr : a->dg; r.bytes[3] = p.value_heads * 4;
  return zero_unowned(p, r, st);
}

}  // namespace la
}  // namespace pkda

extern "C" {

int pkda_la_recurrent_fwd(const pkda_la_recurrent_args* args, void* cuda_stream) {
  if (!args) return PKDA_ERR_NULL;
  pkda::reset_launch_count();
  return pkda::la::recurrent_forward(args, static_cast<cudaStream_t>(cuda_stream));
}
size_t pkda_la_saved_bytes(const pkda_la_problem* p) { return p ? pkda::la::saved_bytes(*p) : 0; }
size_t pkda_la_fwd_workspace_bytes(const pkda_la_problem* p) { return p ? pkda::la::fwd_workspace(*p) : 0; }
int pkda_la_fwd(const pkda_la_fwd_args* args, void* cuda_stream) {
  if (!args) return PKDA_ERR_NULL;
  pkda::reset_launch_count();
  return pkda::la::forward(args, static_cast<cudaStream_t>(cuda_stream));
}
size_t pkda_la_bwd_workspace_bytes(const pkda_la_problem* p) { return p ? pkda::la::bwd_workspace(*p) : 0; }
int pkda_la_bwd(const pkda_la_bwd_args* args, void* cuda_stream) {
  if (!args) return PKDA_ERR_NULL;
  pkda::reset_launch_count();
  return pkda::la::backward(args, static_cast<cudaStream_t>(cuda_stream));
}
size_t pkda_sizeof_la_problem(void) { return sizeof(pkda_la_problem); }
size_t pkda_sizeof_la_recurrent_args(void) { return sizeof(pkda_la_recurrent_args); }
size_t pkda_sizeof_la_fwd_args(void) { return sizeof(pkda_la_fwd_args); }
size_t pkda_sizeof_la_bwd_args(void) { return sizeof(pkda_la_bwd_args); }

}  // extern "C"
