// bst_scan.cuh — what the selective scan's forward and backward kernels share.
//
// Per channel c with N states (arithmetic in fp32):
//   d_t = softplus(delta_t + delta_bias),  a_t[n] = exp(d_t A[n]),
//   h_t[n] = a_t[n] h_{t-1}[n] + d_t u_t B_t[n],   y_t = (sum_n C_t[n] h_t[n] + D u_t) silu(z_t)
//
// Work split: lane = (channel pair, state group).  A warp holds 32 / GS pairs of neighbouring channels
// times GS groups of S states, each lane 2 S of the recurrences, paired over the two channels for the
// two-lane fp32 instructions; it steps through the sequence in order.  Sequences come in tiles of 16
// steps: a block loads a tile of u, delta (z, dy) for its channels and of B, C, computes what is shared
// by the states (the step size) once, and leaves it in shared memory as the steps want it.
#pragma once
#include "bst_layer.cuh"

namespace bst {

constexpr int kScanTile = 16;  // steps per tile, and between two saved states

struct ScanArgs {
  const void *u, *delta, *z, *B, *C, *dy;
  const float *A, *D, *dbias, *init, *dfinal;
  const int* lengths;
  void *y, *du, *ddelta, *dz, *dB, *dC;
  float *final_state, *saved, *dinit;
  float *seg_state, *seg_sum;    // [batch][segments][channels][NP] and [batch][segments][channels]
  float *part_bc;                // [batch][groups][tiles of channels][length][2 NP]
  float *part_a, *part_d;        // [batch][segments][channels][NP], [batch][segments][channels][2]
  int64_t ub, us, db, ds, zb, zs, yb, ys, dyb, dys, Bb, Bs, Bg, Cb, Cs, Cg;
  int64_t length;
  int channels, per_group, groups, states, batch;
  int softplus, vec;
  int segments, seg_tiles, col_tiles;  // segments per sequence, 16-step tiles per segment, channel tiles per group
};

// log2-sized geometry of a warp's work.
template <int S_, int GS_, int W_>
struct ScanShape {
  static constexpr int S = S_, GS = GS_, W = W_;
  static constexpr int NP = S * GS;      // states, padded
  static constexpr int PW = 32 / GS;     // channel pairs per warp
  static constexpr int CT = 2 * PW * W;  // channels per block
  static constexpr int NT = 32 * W;
};

__device__ __forceinline__ int64_t scan_length(const ScanArgs& a, int64_t b) {
  if (!a.lengths) return a.length;
  const int64_t n = a.lengths[b];
  return n < 0 ? 0 : (n < a.length ? n : a.length);
}

// Where a block works.
struct ScanWhere {
  int64_t b;
  int seg, g, ct;
};
__device__ __forceinline__ ScanWhere scan_where(const ScanArgs& a) {
  ScanWhere w;
  int64_t i = blockIdx.x;
  w.ct = int(i % a.col_tiles);
  i /= a.col_tiles;
  w.g = int(i % a.groups);
  i /= a.groups;
  w.seg = int(i % a.segments);
  w.b = i / a.segments;
  return w;
}

// A thread's share of a [16 x CT] tile of an activation: CNT chunks of V elements, chunk i at row
// row(i), column col (the same for all of them).
template <typename T, class Sh>
struct TileShare {
  static constexpr int E = kScanTile * Sh::CT / Sh::NT;  // = PW
  static constexpr int VMAX = 16 / int(sizeof(T));
  static constexpr int V = E < VMAX ? E : VMAX;
  static constexpr int CNT = E / V;
  static constexpr int PER_ROW = Sh::CT / V;
  static constexpr int ROWS = Sh::NT / PER_ROW;  // rows covered by one round of the block
  static_assert(Sh::NT % PER_ROW == 0 && ROWS * CNT == kScanTile, "a round covers whole rows");
  __device__ static int row(int i) { return i * ROWS + int(threadIdx.x) / PER_ROW; }
  __device__ static int col() { return (int(threadIdx.x) % PER_ROW) * V; }
};

// a_t of both channels of a pair; a2 = A log2(e).
__device__ __forceinline__ float2 decay(float2 step, float2 a2) { return ex2_2(mul2(step, a2)); }

// Host: states per lane and the group count for N states.
inline int scan_pad(int64_t n) {
  int p = 4;
  while (p < n) p *= 2;
  return p;
}

int scan_check(const bst_scan_desc* d);
ScanArgs scan_args(const bst_scan_desc* d);
int64_t scan_saved_bytes(const bst_scan_desc* d);
int scan_segments(const bst_scan_desc* d, bool backward, int* tiles);

}  // namespace bst
