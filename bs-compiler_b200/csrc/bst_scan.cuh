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
// steps: a block copies a tile of u, delta (z, dy) for its channels and of B, C into shared memory as they
// are, and computes what is shared by the states (the step size) once.  No store to shared memory stands
// between the steps' loads: the loads of later steps would wait behind it.
#pragma once
#include <cuda.h>
#include <cudaTypedefs.h>

#include <type_traits>

#include "bst_kernels.cuh"  // mbarrier helpers
#include "bst_layer.cuh"

namespace bst {

constexpr int kScanTile = 16;  // steps per tile, and between two saved states

struct ScanArgs {
  const void *u, *delta, *z, *B, *C, *dy;
  const float *A, *D, *dbias, *init, *dfinal;
  const int* lengths;
  void *y, *du, *ddelta, *dz, *dB, *dC;
  float *final_state, *saved, *dinit;
  float *part_bc;                // [batch][groups][tiles of channels][length][2 NP]
  float *part_a, *part_d;        // [batch][channels][NP], [batch][channels][2]
  int64_t ub, us, db, ds, zb, zs, yb, ys, dyb, dys, Bb, Bs, Bg, Cb, Cs, Cg;
  int64_t length;
  int channels, per_group, groups, states, batch;
  int softplus, vec;
  int mode;         // CopyMode of the inputs
  unsigned* error;  // the device's error word
  int col_tiles;    // channel tiles per group
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
  int g, ct;
};
__device__ __forceinline__ ScanWhere scan_where(const ScanArgs& a) {
  ScanWhere w;
  int64_t i = blockIdx.x;
  w.ct = int(i % a.col_tiles);
  i /= a.col_tiles;
  w.g = int(i % a.groups);
  w.b = i / a.groups;
  return w;
}

// A helper thread's share of a [16 x CT] tile: pairs of neighbouring channels, lane by lane along a row, so that
// its accesses to shared memory and to the outputs are contiguous across a warp.  TURNS rows per thread, ROWS apart.
// A block has as many helper threads as recurrence threads; they come second.
template <class Sh>
struct PairShare {
  static constexpr int PAIRS = Sh::CT / 2;
  static constexpr int ROWS = Sh::NT / PAIRS;
  static constexpr int TURNS = kScanTile / ROWS;
  static_assert(Sh::NT % PAIRS == 0 && ROWS * TURNS == kScanTile, "a turn covers whole rows");
  __device__ static int me() { return int(threadIdx.x) - Sh::NT; }
  __device__ static int row(int i) { return i * ROWS + me() / PAIRS; }
  __device__ static int col() { return me() % PAIRS * 2; }
};

// Barriers of a block's two halves, two of each (one per buffer): one half arrives, the other waits.  Their numbers
// are immediates, so that the block does not reserve all sixteen.
enum ScanBarrier : int { kFull = 1, kDone = 3, kHelp = 5 };  // kHelp: among the helpers
template <int THREADS, int ID>
__device__ __forceinline__ void bar_sync(int buf) {
  if (buf) asm volatile("bar.sync %0, %1;" ::"n"(ID + 1), "n"(THREADS) : "memory");
  else asm volatile("bar.sync %0, %1;" ::"n"(ID), "n"(THREADS) : "memory");
}
template <int THREADS, int ID>
__device__ __forceinline__ void bar_arrive(int buf) {
  if (buf) asm volatile("bar.arrive %0, %1;" ::"n"(ID + 1), "n"(THREADS) : "memory");
  else asm volatile("bar.arrive %0, %1;" ::"n"(ID), "n"(THREADS) : "memory");
}

// ---- asynchronous copies of a tile's inputs ------------------------------------------
// How the inputs can be copied (by the alignment of their bases and strides):
enum CopyMode : int {
  kCopyPlain = 0,  // element by element through registers (2-byte elements at odd distances)
  kCopyWords = 1,  // 4 bytes at a time
  kCopyTiles = 2   // whole tiles, by the tensor copy engine (16-byte alignment)
};

__device__ __forceinline__ void copy_async4(void* to, const void* from) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_u32(to)), "l"(from) : "memory");
}
// The inputs as the tensor copy engine sees them: [batch, length, channels] in boxes of 16 positions, and
// [batch, length, groups, states].  What lies outside of a tensor reads zero.
struct ScanMaps {
  CUtensorMap u, delta, z, dy, B, C;
};
__device__ __forceinline__ void tma_load_4d(void* dst, const CUtensorMap* map, uint64_t* bar, int c0, int c1, int c2,
                                            int c3) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(smem_u32(bar))
      : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int LEFT>
__device__ __forceinline__ void copy_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(LEFT) : "memory");
}

// S consecutive floats, as pairs.
template <int S>
struct alignas(4 * S) Pairs {
  float2 v[S / 2];
};
// The first `cols` columns of `rows` rows of a [16 x WIDTH] tile, from rows `step` apart, by NT threads of which this
// one is `me`, in words or elements.  The other columns are filled with zeros, the other rows left as they were.
template <typename T, int WIDTH, int NT>
__device__ __forceinline__ void stage_tile(T* to, const T* from, int64_t step, int rows, int cols, bool words, int me) {
  if (words) {
    constexpr int P = 4 / int(sizeof(T)), ACROSS = WIDTH / P, ITEMS = kScanTile * ACROSS;
#pragma unroll
    for (int i = 0; i < (ITEMS + NT - 1) / NT; ++i) {
      const int k = me + i * NT, r = k / ACROSS, c = k % ACROSS * P;
      if (r < rows) {
        if (c < cols) copy_async4(to + r * WIDTH + c, from + r * step + c);
        else *reinterpret_cast<uint32_t*>(to + r * WIDTH + c) = 0;
      }
    }
  } else {
    constexpr int ITEMS = kScanTile * WIDTH, N = (ITEMS + NT - 1) / NT;
    T v[N];  // all loads before the first store
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int k = me + i * NT, r = k / WIDTH, c = k % WIDTH;
      v[i] = from_f<T>(0.f);
      if (r < rows && c < cols) v[i] = from[r * step + c];
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int k = me + i * NT;
      if (k / WIDTH < rows) to[k] = v[i];
    }
  }
}

// S states of a tile of B or C, as fp32 pairs.
template <int S, typename T>
__device__ __forceinline__ Pairs<S> load_states(const T* p) {
  const Chunk<T, S> c = *reinterpret_cast<const Chunk<T, S>*>(p);
  Pairs<S> r;
#pragma unroll
  for (int i = 0; i < S / 2; ++i) r.v[i] = make_float2(to_f(c.v[2 * i]), to_f(c.v[2 * i + 1]));
  return r;
}

template <typename T>
__device__ __forceinline__ float2 load_pair(const T* p) {
  const Chunk<T, 2> c = *reinterpret_cast<const Chunk<T, 2>*>(p);
  return make_float2(to_f(c.v[0]), to_f(c.v[1]));
}
template <typename T>
__device__ __forceinline__ Chunk<T, 2> to_pair(float2 v) {
  Chunk<T, 2> c;
  c.v[0] = from_f<T>(v.x);
  c.v[1] = from_f<T>(v.y);
  return c;
}

// a_t = 2^x of two states, x = d A log2(e).  The special-function unit's 2^x is good to 2^-22.5; where a_t is near 1 a
// state remembers 1 / (1 - a_t) steps and gathers as many of those errors (the gradient of A lost a digit to it), so
// |x| < 1/16 takes the power series of e^t, t = x ln 2, |t| < 0.0434, up to t^4 / 24 (the rest is below t^5 / 120 =
// 1.3e-9): its one rounding at 1 is that of the last fused operation.
__device__ __forceinline__ float2 decay(float2 step, float2 a2) {
  const float2 x = mul2(step, a2), m = ex2_2(x);
  constexpr float c1 = kLn2, c2 = kLn2 * kLn2 / 2, c3 = kLn2 * kLn2 * kLn2 / 6, c4 = kLn2 * kLn2 * kLn2 * kLn2 / 24;
  float2 p = fma2(both(c4), x, both(c3));
  p = fma2(p, x, both(c2));
  p = fma2(p, x, both(c1));
  p = fma2(p, x, both(1.f));
  return make_float2(fabsf(x.x) < 0.0625f ? p.x : m.x, fabsf(x.y) < 0.0625f ? p.y : m.y);
}

// N states padded to what the lanes of a channel hold.
inline int scan_pad(int64_t n) {
  int p = 4;
  while (p < n) p *= 2;
  return p;
}

int scan_copy_mode(const bst_scan_desc* d, const void* u, const void* delta, const void* z, const void* dy,
                   const void* B, const void* C);
// Tensor maps of a scan's inputs; false where they cannot be made (the words path then copies).
bool scan_maps(const bst_scan_desc* d, int tile_channels, int pad, const void* u, const void* delta, const void* z,
               const void* dy, const void* B, const void* C, ScanMaps* m);

int scan_check(const bst_scan_desc* d);
ScanArgs scan_args(const bst_scan_desc* d);
int64_t scan_saved_bytes(const bst_scan_desc* d);

}  // namespace bst
