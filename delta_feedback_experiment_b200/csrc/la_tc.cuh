// Linear attention in chunks of 64 tokens on tcgen05 (bf16, heads of 128 or 64 channels): what the host side passes to the kernels.
#pragma once

#include "gdr_tc.cuh"
#include "la_common.cuh"

namespace pkda {
namespace la {

// One operation of a launch (la_common.cuh) and the states that go with it.  A CTA takes all segments of a sequence one after the
// other (walk), or one, from a state that is there.
struct ChunkPass {
  Pass p;
  int map[4];             // tensor maps of x, y, z, u
  int reads;              // the gate's gradient: row sums of what is read of R (slices of dots; u: what belongs to out)
  int pairs;              // the gate's gradient: the pairs inside the chunks (backwards; u: the tensor of z's pair products, x y and u z)
  int walk;
  int states_only;        // nothing but R at the segments' ends, from zero, and their decays: what combine_states puts together
  const float* starts;    // [entries][heads] key-major states (not walk): a segment starts from its predecessor's (in time)
  float* ends;            // [entries][heads]: where R goes at the end of a segment, or NULL
  const float* X_states;  // [entries][heads] states at the segments' ends; X = <that, R> at the segment's start in (reversed) time
  float* X;               // [entries][heads][kXParts]
  int* grows;             // [entries][heads]: whether a segment has a decay above 1 (reads; or NULL)
  double* decay;          // [entries][heads] (states_only): the segments' decays, in units of log 2
};
constexpr int kXParts = 8;  // a warp of the state each

struct ChunkCall {
  Call c;
  Segments segments;
  int D;
  int* status;
  const int* order;         // or NULL: the sequences in the order in which walks take them up
  int n;                    // operations
  ChunkPass pass[3];
  const void* base[4];      // tensors of the maps and their heads
  int heads[4];
};

int launch_chunks(const ChunkCall& a, cudaStream_t st);
// The sequences of a packed batch by their chunks, the longest first (all of 255 chunks and more alike; among equals any order, which
// changes no result), so that the last CTAs of a launch are short ones.
int launch_order(const int* bounds, int n_seqs, int* order, cudaStream_t st);
// Slices of Pass::dots that `reads` and `pairs` leave.
__host__ __device__ constexpr int read_slices(int D) { return D / 32; }
constexpr int kPairSlices = 6;

// What states_only left becomes the states that the segments end with: R = init; for all segments in the direction of time,
// R = decay R + entry, entry = R.
int combine_states(const Call& c, const Segments& s, int D, int reverse, const float* init, float* states, const double* decay, cudaStream_t st);

}  // namespace la
}  // namespace pkda
