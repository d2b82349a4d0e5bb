// bst_scan.cuh — what the selective scan's forward and backward kernels share.
//
// Per channel c with N states (arithmetic in fp32):
//   d_t = softplus(delta_t + delta_bias),  a_t[n] = exp(d_t A[n]),
//   h_t[n] = a_t[n] h_{t-1}[n] + d_t u_t B_t[n],   y_t = (sum_n C_t[n] h_t[n] + D u_t) silu(z_t)
//
// Work split: lane = (channels, state group).  A warp holds 32 / GS times CH neighbouring channels times
// GS groups of S states, each lane CH S of the recurrences; neighbouring states are paired for the two-lane
// fp32 instructions, whose B and C operands then lie in shared memory as they are, while the two numbers of
// a channel (d and d u) are doubled in registers: a shared-memory load costs by the bytes that its lanes
// receive, broadcast or not.  A warp steps through the sequence in order.  Sequences come in tiles of 16
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
  int mode_act, mode_bc;  // CopyMode of the activations, of B and C
  int segments, seg_tiles, col_tiles;  // segments per sequence, 16-step tiles per segment, channel tiles per group
};

// Geometry of a block's work: S states and CH channels per lane, GS lanes per channel, W warps.
template <int S_, int CH_, int GS_, int W_>
struct ScanShape {
  static constexpr int S = S_, CH = CH_, GS = GS_, W = W_;
  static constexpr int NP = S * GS;           // states, padded
  static constexpr int CW = CH * (32 / GS);   // channels per warp
  static constexpr int CT = CW * W;           // channels per block
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
  static constexpr int E = kScanTile * Sh::CT / Sh::NT;
  static constexpr int VMAX = 16 / int(sizeof(T));
  static constexpr int V = E < VMAX ? E : VMAX;
  static constexpr int CNT = E / V;
  static constexpr int PER_ROW = Sh::CT / V;
  static constexpr int ROWS = Sh::NT / PER_ROW;  // rows covered by one round of the block
  static_assert(Sh::NT % PER_ROW == 0 && ROWS * CNT == kScanTile, "a round covers whole rows");
  __device__ static int row(int i) { return i * ROWS + int(threadIdx.x) / PER_ROW; }
  __device__ static int col() { return (int(threadIdx.x) % PER_ROW) * V; }
};

// ---- asynchronous copies of a tile's inputs ------------------------------------------
// Each thread copies its own share of a tile into slots of shared memory that only it reads, so that a
// wait for its own copies is all the ordering they need.  How a tensor can be copied:
enum CopyMode : int {
  kCopyPlain = 0,  // element by element through registers (2-byte elements at odd distances)
  kCopyWords = 1,  // 4 bytes at a time
  kCopyChunk = 2   // whole chunks
};

template <int BYTES>
__device__ __forceinline__ void copy_async(void* to, const void* from, bool on) {
  const unsigned dst = unsigned(__cvta_generic_to_shared(to));
  const int n = on ? BYTES : 0;  // the rest of the destination is filled with zeros
  if constexpr (BYTES == 16)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(from), "r"(n) : "memory");
  else
    asm volatile("cp.async.ca.shared.global [%0], [%1], %3, %2;" ::"r"(dst), "l"(from), "r"(n), "n"(BYTES) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int LEFT>
__device__ __forceinline__ void copy_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(LEFT) : "memory");
}

// Elements [0, n) of src (the others zero) into a chunk of shared memory.  `base`: any valid address.
template <typename T, int V>
__device__ __forceinline__ void stage_chunk(Chunk<T, V>* dst, const T* src, const T* base, int n, int mode) {
  constexpr int BYTES = int(sizeof(T)) * V, PER = 4 / int(sizeof(T));
  if constexpr (BYTES >= 4) {
    if (mode == kCopyChunk) {
      copy_async<BYTES>(dst, n >= V ? src : base, n >= V);
      return;
    }
    if (mode == kCopyWords) {
#pragma unroll
      for (int j = 0; j < V; j += PER) copy_async<4>(&dst->v[j], j < n ? src + j : base, j < n);
      return;
    }
  }
#pragma unroll
  for (int j = 0; j < V; ++j) dst->v[j] = j < n ? src[j] : from_f<T>(0.f);
}

// B and C of a tile: pairs of neighbouring states (single ones in fp32), BC of them per thread.
template <typename T, class Sh>
struct StateShare {
  static constexpr int V = 4 / int(sizeof(T));
  static constexpr int ITEMS = kScanTile * Sh::NP / V;
  static constexpr int CNT = (ITEMS + Sh::NT - 1) / Sh::NT;
  __device__ static int item(int i) { return int(threadIdx.x) + i * Sh::NT; }
  __device__ static int row(int k) { return k / (Sh::NP / V); }
  __device__ static int state(int k) { return k % (Sh::NP / V) * V; }
};

// a_t of two states; a2 = A log2(e).
__device__ __forceinline__ float2 decay(float2 step, float2 a2) { return ex2_2(mul2(step, a2)); }

// S consecutive floats, as pairs.
template <int S>
struct alignas(4 * S) Pairs {
  float2 v[S / 2];
};
// What the states of CH neighbouring channels share at one step.
template <int CH>
struct alignas(8 * CH) Step {
  float d[CH], du[CH];
};

// Step sizes d and d u of a thread's chunk of V channels, into the tile's shared memory.
template <int CH, int V>
__device__ __forceinline__ void put_steps(Step<CH>* row, int col, const float (&d)[V], const float (&du)[V]) {
#pragma unroll
  for (int j = 0; j < V; ++j) {
    if constexpr (CH == 2 && V % 2 == 0) {
      if (j % 2 == 0) {
        Step<2> s;
        s.d[0] = d[j], s.d[1] = d[j + 1], s.du[0] = du[j], s.du[1] = du[j + 1];
        row[(col + j) / 2] = s;
      }
    } else {
      row[(col + j) / CH].d[(col + j) % CH] = d[j];
      row[(col + j) / CH].du[(col + j) % CH] = du[j];
    }
  }
}

// v -> f2 of neighbouring values (f1 of a single one).
template <int V, class F1, class F2>
__device__ __forceinline__ void by_two(float (&v)[V], F1&& f1, F2&& f2) {
  if constexpr (V == 1) {
    v[0] = f1(v[0]);
  } else {
#pragma unroll
    for (int j = 0; j < V; j += 2) {
      const float2 r = f2(make_float2(v[j], v[j + 1]));
      v[j] = r.x;
      v[j + 1] = r.y;
    }
  }
}

// Host: states per lane and the group count for N states.
inline int scan_pad(int64_t n) {
  int p = 4;
  while (p < n) p *= 2;
  return p;
}

// How activations whose base pointers and strides are or-ed into `bits` (in bytes) can be copied.
inline int copy_mode(uint64_t bits) { return bits % 16 == 0 ? kCopyChunk : bits % 4 == 0 ? kCopyWords : kCopyPlain; }

int scan_check(const bst_scan_desc* d);
ScanArgs scan_args(const bst_scan_desc* d);
int64_t scan_saved_bytes(const bst_scan_desc* d);
int scan_segments(const bst_scan_desc* d, bool backward, int* tiles);

}  // namespace bst
