// bst_norm.cu — layer norm, forward and backward (bst_layer_norm_*).
//
// Forward, per row of D entries:  mean = sum x / D,  var = sum (x - mean)^2 / D,
//   rstd = 1 / sqrt(var + eps),  y = (x - mean) rstd w + b.
// Backward, with xh = (x - mean) rstd and g = w dy:
//   dx = rstd (g - sum g / D - xh sum(g xh) / D),   dw = sum_rows dy xh,   db = sum_rows dy.
//
// Both move every element once and do a dozen operations on it, so HBM bounds them: a row is held in
// registers from its only read to its write (the variance is a second sweep over the registers, which
// costs no traffic and does not cancel as E[x^2] - mean^2 would).  The rows of a block's turn are
// `slots`, TPR threads each; a block walks over the rows, so that w and the sums for dw and db stay in
// its threads' registers for the whole pass and leave it once, as one partial row per slot.  A second
// launch adds the partial rows up in a fixed order.
//
// Measured on B200, 16384 x 4096 in bf16 with fp32 parameters: forward 60 us (4.5 TB/s; 75 us with the next row
// prefetched into registers instead of the ring, 164 us with neither), backward 81 us (5.0 TB/s; 110 and 161 us),
// the partial rows' sum 4 us.  A plain copy moves 6.55 TB/s.  Rows of a few hundred bytes and single rows are
// bound by their launch and by the latency of one row (5 x 1541 in fp16, not aligned: 7 us).
#include <algorithm>

#include "bst_kernels.cuh"  // mbarrier helpers
#include "bst_layer.cuh"

namespace bst {

int occupancy(const void* fn, int threads, int smem);  // bst_core.cu

constexpr int kNormItems = 16;        // elements of a row per thread
constexpr int kNormMaxThreads = 1024; // longer rows than 1024 * 16 go through the kernels that re-read

struct NormArgs {
  const void *x, *w, *b, *dy;
  void *y, *dx;
  float *mean, *rstd;             // forward: outputs (may be null)
  const float *mean_in, *rstd_in; // backward
  float* part;                    // [slots][2][dim] partial sums of dw, db
  int64_t rows, xs, ys, dys, dxs;
  int dim, wide, vec, params;     // wide: parameters are fp32; params: dw or db asked for
  float eps, inv_dim;
  int stages;       // of the ring
  unsigned* error;  // the device's error word
};

template <typename T>
__device__ __forceinline__ float param_at(const void* p, int wide, int i) {
  return wide ? static_cast<const float*>(p)[i] : to_f(static_cast<const T*>(p)[i]);
}
// Parameters i .. i + V - 1 (`missing` where there are none).
template <typename T, int V>
__device__ __forceinline__ void load_params(const void* p, int wide, int i, int dim, float missing,
                                            float (&v)[V]) {
  if (!p) {
#pragma unroll
    for (int j = 0; j < V; ++j) v[j] = missing;
  } else if (V > 1 && i < dim) {  // more than one column per access: dim is a multiple of V, all is aligned
    if (wide) {
      const Chunk<float, V < 4 ? V : 4>* q = reinterpret_cast<const Chunk<float, V < 4 ? V : 4>*>(
          static_cast<const float*>(p) + i);
#pragma unroll
      for (int j = 0; j < V; ++j) v[j] = q[j / 4].v[j % 4];
    } else {
      const Chunk<T, V> c = *reinterpret_cast<const Chunk<T, V>*>(static_cast<const T*>(p) + i);
#pragma unroll
      for (int j = 0; j < V; ++j) v[j] = to_f(c.v[j]);
    }
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j) v[j] = i + j < dim ? param_at<T>(p, wide, i + j) : missing;
  }
}

// Sums of v over the TPR threads of a row's slot, known to all of them.  `buf`: two halves of TPR / 32 entries for the
// slot, used in turn (`half`), so that one barrier per sum is enough.
template <int TPR, typename V>
__device__ __forceinline__ V row_sum(V v, V (*buf)[TPR / 32], int& half) {
  constexpr bool TWO = sizeof(V) == sizeof(float2);
  auto lane_sum = [](V x, int m) {
    if constexpr (TWO) {
      x.x += __shfl_xor_sync(0xffffffffu, x.x, m);
      x.y += __shfl_xor_sync(0xffffffffu, x.y, m);
    } else {
      x += __shfl_xor_sync(0xffffffffu, x, m);
    }
    return x;
  };
#pragma unroll
  for (int m = 16; m >= 1; m >>= 1) v = lane_sum(v, m);
  if constexpr (TPR > 32) {
    const int t = threadIdx.x % TPR;
    V* to = buf[half];
    half ^= 1;
    if (t % 32 == 0) to[t / 32] = v;
    __syncthreads();
    v = to[t % (TPR / 32)];
#pragma unroll
    for (int m = TPR / 64; m >= 1; m >>= 1) v = lane_sum(v, m);
  }
  return v;
}

// Rows on their way into shared memory: a ring of STAGES rows of each of N tensors per slot, filled by the bulk copy
// engine (whole rows, 16-byte aligned).  It keeps more bytes under way than the threads' registers could.
constexpr int kNormMaxStages = 4;
constexpr int kNormRingHeader = 256;  // the barriers of up to 8 slots
constexpr int kNormRingMost = 200 * 1024;  // two stages of a block's rows have to fit in shared memory
template <typename T, int N>
struct RowRing {
  T* data;         // [stages][N][dim] of this slot
  uint64_t* bar;   // [stages]
  int dim, stages;
  bool failed;

  __device__ __forceinline__ void start(unsigned char* shared, int n, int slot, int d, bool leader) {
    dim = d;
    stages = n;
    failed = false;
    bar = reinterpret_cast<uint64_t*>(shared) + slot * kNormMaxStages;
    data = reinterpret_cast<T*>(shared + kNormRingHeader) + int64_t(slot) * n * N * d;
    if (leader) {
      for (int i = 0; i < n; ++i) mbar_init(&bar[i], 1);
      mbar_fence_init();
    }
    __syncthreads();
  }
  __device__ __forceinline__ T* row(int stage, int n) const { return data + (stage * N + n) * int64_t(dim); }
  __device__ __forceinline__ void expect(int stage) { mbar_expect_tx(&bar[stage], unsigned(N * dim * sizeof(T))); }
  __device__ __forceinline__ void copy(int stage, int n, const T* from) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                     smem_u32(row(stage, n))),
                 "l"(from), "r"(unsigned(dim * sizeof(T))), "r"(smem_u32(&bar[stage]))
                 : "memory");
  }
  __device__ __forceinline__ void wait(int stage, unsigned parity, unsigned* error) {
    if (!failed && !mbar_wait_bounded(&bar[stage], parity)) {
      failed = true;
      atomicOr(error, kErrTmaTimeout);
    }
  }
};

// First column of chunk k of thread t of a row.
template <int TPR, int V>
__device__ __forceinline__ int column(int t, int k) { return (k * TPR + t) * V; }

// The parameters of a thread's columns stay in its registers.  Rows arrive ahead of their turn: through the ring where
// whole vectors can be read (V > 1), one row ahead in registers otherwise.
template <typename T, int TPR, int V>
__global__ void __launch_bounds__(TPR < 256 ? 256 : TPR, TPR > 512 ? 1 : 768 / (TPR < 256 ? 256 : TPR))
    norm_forward_kernel(const NormArgs a) {
  constexpr int NT = TPR < 256 ? 256 : TPR, SLOTS = NT / TPR, NC = kNormItems / V;
  constexpr bool RING = V > 1;
  __shared__ float buf[SLOTS][2][TPR / 32];
  extern __shared__ __align__(128) unsigned char shared[];
  const int t = threadIdx.x % TPR, slot = threadIdx.x / TPR;
  int half = 0, stage = 0;
  unsigned parity = 0;
  const int64_t stride = int64_t(gridDim.x) * SLOTS;
  int64_t row = int64_t(blockIdx.x) * SLOTS + slot;
  const T* base = static_cast<const T*>(a.x);
  RowRing<T, 1> ring;
  Chunk<T, V> c[NC];
  auto load = [&](int64_t r) {
#pragma unroll
    for (int k = 0; k < NC; ++k) {
      const int i = column<TPR, V>(t, k);
      c[k] = load_whole<T, V>(base + r * a.xs + i, r < a.rows && i < a.dim);
    }
  };
  auto send = [&](int to, int64_t r) {
    if (t == 0 && r < a.rows) {
      ring.expect(to);
      ring.copy(to, 0, base + r * a.xs);
    }
  };
  if constexpr (RING) {
    ring.start(shared, a.stages, slot, a.dim, t == 0);
    for (int i = 0; i < a.stages; ++i) send(i, row + i * stride);
  } else {
    load(row);
  }
  float w[NC][V], b[NC][V];
#pragma unroll
  for (int k = 0; k < NC; ++k) {
    load_params<T, V>(a.w, a.wide, column<TPR, V>(t, k), a.dim, 1.f, w[k]);
    load_params<T, V>(a.b, a.wide, column<TPR, V>(t, k), a.dim, 0.f, b[k]);
  }
  // Every slot of the block makes the same number of turns: the sums hold barriers.
  for (int64_t row0 = int64_t(blockIdx.x) * SLOTS; row0 < a.rows; row0 += stride, row += stride) {
    if constexpr (RING) {
      if (row < a.rows) ring.wait(stage, parity, a.error);
#pragma unroll
      for (int k = 0; k < NC; ++k) {
        const int i = column<TPR, V>(t, k);
        c[k] = load_whole<T, V>(ring.row(stage, 0) + i, row < a.rows && i < a.dim);
      }
    }
    float x[NC][V], s = 0.f, q = 0.f;
#pragma unroll
    for (int k = 0; k < NC; ++k)
#pragma unroll
      for (int j = 0; j < V; ++j) s += x[k][j] = to_f(c[k].v[j]);
    if constexpr (!RING) load(row + stride);
    const float mean = row_sum<TPR>(s, buf[slot], half) * a.inv_dim;
    if constexpr (RING) {  // everybody has read the row: its place is free
      if (TPR == 32) __syncwarp();
      send(stage, row + a.stages * stride);
      if (++stage == a.stages) stage = 0, parity ^= 1;
    }
#pragma unroll
    for (int k = 0; k < NC; ++k)
#pragma unroll
      for (int j = 0; j < V; ++j) {
        x[k][j] = column<TPR, V>(t, k) + j < a.dim ? x[k][j] - mean : 0.f;
        q = fmaf(x[k][j], x[k][j], q);
      }
    const float var = row_sum<TPR>(q, buf[slot], half) * a.inv_dim;
    const float rstd = 1.f / sqrtf(var + a.eps);
    if (row >= a.rows) continue;
    if (t == 0) {
      if (a.mean) a.mean[row] = mean;
      if (a.rstd) a.rstd[row] = rstd;
    }
    T* y = static_cast<T*>(a.y) + row * a.ys;
#pragma unroll
    for (int k = 0; k < NC; ++k) {
      Chunk<T, V> o;
#pragma unroll
      for (int j = 0; j < V; ++j) o.v[j] = from_f<T>(fmaf(x[k][j] * rstd, w[k][j], b[k][j]));
      const int i = column<TPR, V>(t, k);
      store_whole<T, V>(y + i, o, i < a.dim);
    }
  }
  if (RING && ring.failed)  // a row that is late may not outlive the block
    for (int i = 0; i < a.stages; ++i) mbar_wait_bounded(&ring.bar[i], parity);
}

template <typename T, int TPR, int V>
__global__ void __launch_bounds__(TPR < 256 ? 256 : TPR, TPR > 256 ? 1 : 2) norm_backward_kernel(const NormArgs a) {
  constexpr int NT = TPR < 256 ? 256 : TPR, SLOTS = NT / TPR, NC = kNormItems / V;
  constexpr bool RING = V > 1;
  __shared__ float2 buf[SLOTS][2][TPR / 32];
  extern __shared__ __align__(128) unsigned char shared[];
  const int t = threadIdx.x % TPR, slot = threadIdx.x / TPR;
  int half = 0, stage = 0;
  unsigned parity = 0;
  const int64_t stride = int64_t(gridDim.x) * SLOTS;
  int64_t row = int64_t(blockIdx.x) * SLOTS + slot;
  RowRing<T, 2> ring;
  Chunk<T, V> nx[NC], nd[NC];
  float next_mean = 0.f, next_rstd = 0.f;
  auto load = [&](int64_t r) {
    const bool live = r < a.rows;
    const T* x = static_cast<const T*>(a.x) + r * a.xs;
    const T* dy = static_cast<const T*>(a.dy) + r * a.dys;
#pragma unroll
    for (int k = 0; k < NC; ++k) {
      const int i = column<TPR, V>(t, k);
      nx[k] = load_whole<T, V>(x + i, live && i < a.dim);
      nd[k] = load_whole<T, V>(dy + i, live && i < a.dim);
    }
    next_mean = live ? a.mean_in[r] : 0.f;
    next_rstd = live ? a.rstd_in[r] : 0.f;
  };
  auto send = [&](int to, int64_t r) {
    if (t == 0 && r < a.rows) {
      ring.expect(to);
      ring.copy(to, 0, static_cast<const T*>(a.x) + r * a.xs);
      ring.copy(to, 1, static_cast<const T*>(a.dy) + r * a.dys);
    }
  };
  if constexpr (RING) {
    ring.start(shared, a.stages, slot, a.dim, t == 0);
    for (int i = 0; i < a.stages; ++i) send(i, row + i * stride);
    next_mean = row < a.rows ? a.mean_in[row] : 0.f;
    next_rstd = row < a.rows ? a.rstd_in[row] : 0.f;
  } else {
    load(row);
  }
  float w[NC][V], dw[NC][V], db[NC][V];
#pragma unroll
  for (int k = 0; k < NC; ++k) {
    load_params<T, V>(a.w, a.wide, column<TPR, V>(t, k), a.dim, 1.f, w[k]);
#pragma unroll
    for (int j = 0; j < V; ++j) dw[k][j] = db[k][j] = 0.f;
  }
  for (int64_t row0 = int64_t(blockIdx.x) * SLOTS; row0 < a.rows; row0 += stride, row += stride) {
    Chunk<T, V> cx[NC], cd[NC];
    const float mean = next_mean, rstd = next_rstd;
    if constexpr (RING) {
      const bool live = row < a.rows, more = row + stride < a.rows;
      if (live) ring.wait(stage, parity, a.error);
      next_mean = more ? a.mean_in[row + stride] : 0.f;
      next_rstd = more ? a.rstd_in[row + stride] : 0.f;
#pragma unroll
      for (int k = 0; k < NC; ++k) {
        const int i = column<TPR, V>(t, k);
        cx[k] = load_whole<T, V>(ring.row(stage, 0) + i, live && i < a.dim);
        cd[k] = load_whole<T, V>(ring.row(stage, 1) + i, live && i < a.dim);
      }
    } else {
#pragma unroll
      for (int k = 0; k < NC; ++k) cx[k] = nx[k], cd[k] = nd[k];
      if (row0 + stride < a.rows) load(row + stride);
    }
    float2 s = make_float2(0.f, 0.f);
#pragma unroll
    for (int k = 0; k < NC; ++k)
#pragma unroll
      for (int j = 0; j < V; ++j) {
        // Columns beyond dim hold dy = 0.
        const float d = to_f(cd[k].v[j]);
        const float xh = (to_f(cx[k].v[j]) - mean) * rstd;
        const float g = d * w[k][j];
        s.x += g;
        s.y = fmaf(g, xh, s.y);
        dw[k][j] = fmaf(d, xh, dw[k][j]);
        db[k][j] += d;
      }
    s = row_sum<TPR>(s, buf[slot], half);
    if constexpr (RING) {  // everybody has read the row: its place is free
      if (TPR == 32) __syncwarp();
      send(stage, row + a.stages * stride);
      if (++stage == a.stages) stage = 0, parity ^= 1;
    }
    const float m1 = s.x * a.inv_dim, m2 = s.y * a.inv_dim;
    if (row >= a.rows) continue;
    T* dx = static_cast<T*>(a.dx) + row * a.dxs;
#pragma unroll
    for (int k = 0; k < NC; ++k) {
      const int i = column<TPR, V>(t, k);
      Chunk<T, V> o;
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float xh = (to_f(cx[k].v[j]) - mean) * rstd;
        o.v[j] = from_f<T>(rstd * (to_f(cd[k].v[j]) * w[k][j] - m1 - xh * m2));
      }
      store_whole<T, V>(dx + i, o, i < a.dim);
    }
  }
  if (RING && ring.failed)  // a row that is late may not outlive the block
    for (int i = 0; i < a.stages; ++i) mbar_wait_bounded(&ring.bar[i], parity);
  if (!a.params) return;
  float* p = a.part + (int64_t(blockIdx.x) * SLOTS + slot) * 2 * a.dim;
#pragma unroll
  for (int k = 0; k < NC; ++k)
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int i = column<TPR, V>(t, k) + j;
      if (i < a.dim) {
        p[i] = dw[k][j];
        p[a.dim + i] = db[k][j];
      }
    }
}

// ---- rows too long for a block's registers: the row is read again for each sum ------------
template <typename T>
__global__ void __launch_bounds__(1024) norm_forward_long_kernel(const NormArgs a) {
  __shared__ float buf[2][32];
  int half = 0;
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T* x = static_cast<const T*>(a.x) + row * a.xs;
    T* y = static_cast<T*>(a.y) + row * a.ys;
    float s = 0.f, q = 0.f;
    for (int i = threadIdx.x; i < a.dim; i += 1024) s += to_f(x[i]);
    const float mean = row_sum<1024>(s, buf, half) * a.inv_dim;
    for (int i = threadIdx.x; i < a.dim; i += 1024) {
      const float d = to_f(x[i]) - mean;
      q = fmaf(d, d, q);
    }
    const float rstd = 1.f / sqrtf(row_sum<1024>(q, buf, half) * a.inv_dim + a.eps);
    if (threadIdx.x == 0) {
      if (a.mean) a.mean[row] = mean;
      if (a.rstd) a.rstd[row] = rstd;
    }
    for (int i = threadIdx.x; i < a.dim; i += 1024) {
      const float w = a.w ? param_at<T>(a.w, a.wide, i) : 1.f, b = a.b ? param_at<T>(a.b, a.wide, i) : 0.f;
      y[i] = from_f<T>(fmaf((to_f(x[i]) - mean) * rstd, w, b));
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(1024) norm_backward_long_kernel(const NormArgs a) {
  __shared__ float2 buf[2][32];
  int half = 0;
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T* x = static_cast<const T*>(a.x) + row * a.xs;
    const T* dy = static_cast<const T*>(a.dy) + row * a.dys;
    T* dx = static_cast<T*>(a.dx) + row * a.dxs;
    const float mean = a.mean_in[row], rstd = a.rstd_in[row];
    float2 s = make_float2(0.f, 0.f);
    for (int i = threadIdx.x; i < a.dim; i += 1024) {
      const float g = to_f(dy[i]) * (a.w ? param_at<T>(a.w, a.wide, i) : 1.f);
      s.x += g;
      s.y = fmaf(g, (to_f(x[i]) - mean) * rstd, s.y);
    }
    s = row_sum<1024>(s, buf, half);
    const float m1 = s.x * a.inv_dim, m2 = s.y * a.inv_dim;
    for (int i = threadIdx.x; i < a.dim; i += 1024) {
      const float g = to_f(dy[i]) * (a.w ? param_at<T>(a.w, a.wide, i) : 1.f);
      dx[i] = from_f<T>(rstd * (g - m1 - (to_f(x[i]) - mean) * rstd * m2));
    }
  }
}

// Partial rows of dw and db for those: blockIdx.y takes every gridDim.y-th row.
template <typename T>
__global__ void __launch_bounds__(256) norm_params_long_kernel(const NormArgs a) {
  const int i = blockIdx.x * 256 + threadIdx.x;
  if (i >= a.dim) return;
  float dw = 0.f, db = 0.f;
  for (int64_t row = blockIdx.y; row < a.rows; row += gridDim.y) {
    const float d = to_f(static_cast<const T*>(a.dy)[row * a.dys + i]);
    dw = fmaf(d, (to_f(static_cast<const T*>(a.x)[row * a.xs + i]) - a.mean_in[row]) * a.rstd_in[row], dw);
    db += d;
  }
  float* p = a.part + int64_t(blockIdx.y) * 2 * a.dim;
  p[i] = dw;
  p[a.dim + i] = db;
}

// dw, db = sums of `slots` partial rows of 2 * dim values.  32 columns a block, 32 threads a column.
template <typename P>
__global__ void __launch_bounds__(1024) norm_params_kernel(const float* part, int64_t slots, int dim, P* dw, P* db) {
  __shared__ float sums[32][33];
  const int c = threadIdx.x % 32, r = threadIdx.x / 32;
  const int64_t i = int64_t(blockIdx.x) * 32 + c, n = 2 * int64_t(dim);
  float s = 0.f;
  if (i < n) {
    int64_t k = r;
    for (; k + 7 * 32 < slots; k += 8 * 32) {  // loads in flight together, added in order
      float v[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = part[(k + j * 32) * n + i];
#pragma unroll
      for (int j = 0; j < 8; ++j) s += v[j];
    }
    for (; k < slots; k += 32) s += part[k * n + i];
  }
  sums[r][c] = s;
  __syncthreads();
  s = warp_sum(sums[c][r]);  // warp r now adds up column r of the block
  const int64_t o = int64_t(blockIdx.x) * 32 + r;
  if (c == 0 && o < n) {
    if (o < dim) {
      if (dw) dw[o] = from_f<P>(s);
    } else if (db) {
      db[o - dim] = from_f<P>(s);
    }
  }
}

// Threads per row: the fewest of 32, 128, .. 1024 that hold it (0: none does).
static int norm_threads(int64_t dim) {
  for (int t : {32, 128, 256, 512, kNormMaxThreads})
    if (dim <= int64_t(t) * kNormItems) return t;
  return 0;
}
constexpr int kNormBlocksPerSm = 2;  // of the backward pass (its launch bounds): each slot leaves a partial row

static int64_t norm_backward_blocks(int64_t rows, int tpr) {
  const int slots = tpr < 256 ? 256 / tpr : 1;
  return std::max<int64_t>(1, std::min<int64_t>((rows + slots - 1) / slots, int64_t(sm_count()) * (tpr > 256 ? 1 : kNormBlocksPerSm)));
}
static int64_t norm_slots(const bst_norm_desc* d) {
  const int tpr = norm_threads(d->dim);
  if (tpr == 0) return std::min<int64_t>(std::max<int64_t>(d->rows, 1), 64);
  return norm_backward_blocks(d->rows, tpr) * (tpr < 256 ? 256 / tpr : 1);
}

static int norm_check(const bst_norm_desc* d) {
  if (!d) return fail(BST_ERR_INVALID, "null description");
  if (!layer_dtype(d->dtype)) return fail(BST_ERR_UNSUPPORTED, "layer norm runs in float32, bfloat16 or float16");
  if (d->param_dtype != d->dtype && d->param_dtype != BST_F32)
    return fail(BST_ERR_UNSUPPORTED, "layer norm parameters must have the input's type or float32");
  if (d->rows < 0 || d->dim < 0) return fail(BST_ERR_INVALID, "negative extent");
  if (d->dim > (int64_t(1) << 30)) return fail(BST_ERR_UNSUPPORTED, "rows of more than 2^30 entries");
  if (!(d->eps >= 0)) return fail(BST_ERR_INVALID, "eps must be non-negative");
  return BST_OK;
}

template <typename T, bool BWD>
static int norm_launch(const NormArgs& a, int tpr, int64_t blocks, cudaStream_t st) {
  constexpr int VW = 16 / int(sizeof(T));
  auto go = [&](auto tprc, auto vc) {
    constexpr int TPR = decltype(tprc)::value, V = decltype(vc)::value;
    constexpr int NT = TPR < 256 ? 256 : TPR;
    const int stage = (NT / TPR) * (BWD ? 2 : 1) * a.dim * int(sizeof(T));
    NormArgs args = a;
    args.stages = std::max(2, std::min(kNormMaxStages, 64 * 1024 / stage));
    const int smem = V > 1 ? kNormRingHeader + args.stages * stage : 0;
    // The limit belongs to the kernel, not to the call: every call sets the same one, the most that any needs, so that
    // calls with other row lengths on other threads cannot take this one's room away before its launch.
    const int most_smem = V > 1 ? kNormRingHeader + kNormRingMost : 0;
    if constexpr (BWD) {
      auto* kernel = norm_backward_kernel<T, TPR, V>;
      BST_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, most_smem));
      kernel<<<unsigned(blocks), NT, smem, st>>>(args);
    } else {
      // A block walks over the rows and keeps its parameters: no more of them than are resident.
      auto* kernel = norm_forward_kernel<T, TPR, V>;
      BST_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, most_smem));
      const int64_t most = int64_t(sm_count()) * std::max(1, occupancy((const void*)kernel, NT, smem));
      kernel<<<unsigned(std::min(blocks, most)), NT, smem, st>>>(args);
    }
    return launched(BWD ? "norm_backward_kernel launch" : "norm_forward_kernel launch");
  };
  auto pick = [&](auto tprc) {
    return a.vec ? go(tprc, std::integral_constant<int, VW>{}) : go(tprc, std::integral_constant<int, 1>{});
  };
  switch (tpr) {
    case 32: return pick(std::integral_constant<int, 32>{});
    case 128: return pick(std::integral_constant<int, 128>{});
    case 256: return pick(std::integral_constant<int, 256>{});
    case 512: return pick(std::integral_constant<int, 512>{});
    default: return pick(std::integral_constant<int, 1024>{});
  }
}

}  // namespace bst

using namespace bst;

extern "C" {

int bst_layer_norm_forward(const bst_norm_desc* d, const void* x, const void* weight, const void* bias, void* y,
                           float* mean, float* rstd, void* stream) {
  clear_error();
  if (int rc = norm_check(d)) return rc;
  if (d->rows == 0 || d->dim == 0) return BST_OK;
  if (!x || !y) return fail(BST_ERR_INVALID, "null device pointer");
  const int64_t es = layer_elem_size(d->dtype), per = 16 / es;
  NormArgs a{};
  a.x = x, a.w = weight, a.b = bias, a.y = y, a.mean = mean, a.rstd = rstd;
  a.rows = d->rows, a.xs = d->x_row, a.ys = d->y_row, a.dim = int(d->dim);
  a.wide = d->param_dtype == BST_F32 && d->dtype != BST_F32;
  a.vec = aligned16(x) && aligned16(y) && aligned16(weight) && aligned16(bias) && d->dim % per == 0 && d->x_row % per == 0 && d->y_row % per == 0;
  a.eps = float(d->eps), a.inv_dim = 1.f / float(d->dim);
  a.vec = a.vec && 2 * d->dim * es <= kNormRingMost;
  a.error = device_error_word();
  if (!a.error) return fail(BST_ERR_CUDA, "device error word unavailable");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int tpr = norm_threads(d->dim);
  const int slots = tpr && tpr < 256 ? 256 / tpr : 1;
  const int64_t blocks = (d->rows + slots - 1) / slots;
  return with_type(d->dtype, [&](auto t) {
    using T = decltype(t);
    if (tpr) return norm_launch<T, false>(a, tpr, blocks, st);
    norm_forward_long_kernel<T><<<unsigned(std::min<int64_t>(blocks, INT_MAX)), 1024, 0, st>>>(a);
    return launched("norm_forward_long_kernel launch");
  });
}

int bst_layer_norm_workspace(const bst_norm_desc* d, int64_t* bytes) {
  clear_error();
  if (int rc = norm_check(d)) return rc;
  if (!bytes) return fail(BST_ERR_INVALID, "null output");
  *bytes = d->rows == 0 || d->dim == 0 ? 0 : norm_slots(d) * 2 * d->dim * 4;
  return BST_OK;
}

int bst_layer_norm_backward(const bst_norm_desc* d, const void* x, const void* weight, const void* dy,
                            const float* mean, const float* rstd, void* dx, void* dweight, void* dbias,
                            void* workspace, int64_t workspace_bytes, void* stream) {
  int64_t need = 0;
  if (int rc = bst_layer_norm_workspace(d, &need)) return rc;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int64_t es = layer_elem_size(d->dtype), per = 16 / es, ps = layer_elem_size(d->param_dtype);
  if (d->dim == 0) return BST_OK;
  if (d->rows == 0) {
    if (dweight) BST_CUDA(cudaMemsetAsync(dweight, 0, size_t(d->dim * ps), st));
    if (dbias) BST_CUDA(cudaMemsetAsync(dbias, 0, size_t(d->dim * ps), st));
    return BST_OK;
  }
  if (!x || !dy || !dx || !mean || !rstd) return fail(BST_ERR_INVALID, "null device pointer");
  const bool params = dweight || dbias;
  if (params && (!workspace || workspace_bytes < need || !aligned16(workspace)))
    return fail(BST_ERR_INVALID, "the workspace must hold " + std::to_string(need) + " bytes, aligned to 16");
  NormArgs a{};
  a.x = x, a.w = weight, a.dy = dy, a.dx = dx, a.mean_in = mean, a.rstd_in = rstd;
  a.part = static_cast<float*>(workspace);
  a.rows = d->rows, a.xs = d->x_row, a.dys = d->dy_row, a.dxs = d->dx_row, a.dim = int(d->dim);
  a.wide = d->param_dtype == BST_F32 && d->dtype != BST_F32;
  a.vec = aligned16(x) && aligned16(dy) && aligned16(dx) && aligned16(weight) && d->dim % per == 0 && d->x_row % per == 0 &&
          d->dy_row % per == 0 && d->dx_row % per == 0;
  a.vec = a.vec && 4 * d->dim * es <= kNormRingMost;
  a.params = params;
  a.error = device_error_word();
  if (!a.error) return fail(BST_ERR_CUDA, "device error word unavailable");
  a.inv_dim = 1.f / float(d->dim);
  const int tpr = norm_threads(d->dim);
  int rc = with_type(d->dtype, [&](auto t) {
    using T = decltype(t);
    if (tpr) return norm_launch<T, true>(a, tpr, norm_backward_blocks(d->rows, tpr), st);
    norm_backward_long_kernel<T><<<unsigned(std::min<int64_t>(d->rows, INT_MAX)), 1024, 0, st>>>(a);
    if (int e = launched("norm_backward_long_kernel launch")) return e;
    if (!params) return int(BST_OK);
    norm_params_long_kernel<T><<<dim3(unsigned((d->dim + 255) / 256), unsigned(norm_slots(d))), 256, 0, st>>>(a);
    return launched("norm_params_long_kernel launch");
  });
  if (rc || !params) return rc;
  const unsigned blocks = unsigned((2 * d->dim + 31) / 32);
  return with_type(d->param_dtype, [&](auto t) {
    using P = decltype(t);
    norm_params_kernel<P><<<blocks, 1024, 0, st>>>(a.part, norm_slots(d), a.dim, static_cast<P*>(dweight),
                                                   static_cast<P*>(dbias));
    return launched("norm_params_kernel launch");
  });
}

}  // extern "C"
