// bst_conv.cu — short causal depthwise convolution: forward, backward and single-position step
// (bst_causal_conv_*).
//
//   p[t] = bias + sum_k w[k] x[t - W + 1 + k],   y = p or p sigmoid(p)            (per channel)
//   q[t] = dy[t] (silu: times s + p s (1 - s), s = sigmoid(p))
//   dx[t] = sum_k w[k] q[t + W - 1 - k],   dw[k] = sum_t q[t] x[t - W + 1 + k],   dbias = sum_t q[t]
//
// A handful of operations per element: HBM bounds every pass.  Two layouts:
//  * channels contiguous (`march`): a thread owns a 16-byte vector of channels and marches along the
//    sequence with the last W - 1 inputs in registers, as the 3-D stencil kernels march along Z, so
//    each element is loaded once, and the weights and the sums for dw stay in its registers;
//  * sequence contiguous (`lines`): a block owns a piece of one channel's line and a thread one
//    position; the W - 1 neighbours come out of L1.
// A piece of a sequence reads W - 1 positions of the piece before it (the backward pass also W - 1 of
// the one behind it, whose q it computes again).  Sums for dw and dbias leave each piece as one partial
// row and are added up by a second launch in a fixed order.
//
// Measured on B200, width 4 with silu in bf16: forward 1 x 8192 x 4096 40 us, 4 x 4096 x 4096 69 us (3.9 TB/s of a
// plain copy's 6.55), bound by the loads that its registers can keep under way; backward 4 x 4096 x 4096 155 us
// (2.6 TB/s), bound by instruction issue (the silu's slope and 3 width fused operations per element), its sums 17 us.
#include <algorithm>

#include "bst_layer.cuh"

namespace bst {

struct ConvArgs {
  const void *x, *w, *b, *init, *dy, *dfinal;
  void *y, *final_state, *dx, *dinit;
  const int* lengths;
  float* part;  // [pieces][W + 1][channels] partial sums of dw and dbias
  int64_t xb, xs, yb, ys, dyb, dys, dxb, dxs;
  int64_t length;
  int channels, wide, vec, silu;
  int pieces, piece;  // pieces per sequence, positions per piece
};

template <typename T>
__device__ __forceinline__ float conv_param(const void* p, int wide, int64_t i) {
  return wide ? static_cast<const float*>(p)[i] : to_f(static_cast<const T*>(p)[i]);
}
__device__ __forceinline__ int64_t live_length(const int* lengths, int64_t length, int64_t b) {
  if (!lengths) return length;
  const int64_t n = lengths[b];
  return n < 0 ? 0 : (n < length ? n : length);
}
// q / dy: the derivative of y with respect to p.
__device__ __forceinline__ float silu_slope(float p) {
  const float s = sigmoid(p);
  return s * fmaf(p, 1.f - s, 1.f);
}

// The input at position t >= -(W - 1) of V channels: of x, or of the initial state.
template <typename T, int V, int W>
__device__ __forceinline__ Chunk<T, V> input_at(const ConvArgs& a, int64_t b, int64_t t, int c) {
  if (t >= 0) return load_whole<T, V>(static_cast<const T*>(a.x) + b * a.xb + t * a.xs + c, true);
  return load_whole<T, V>(static_cast<const T*>(a.init) + (b * (W - 1) + t + W - 1) * a.channels + c, a.init != nullptr);
}

// V channels as pairs (a pair of one where V is 1).
template <int V>
struct Lanes {
  static constexpr int P = (V + 1) / 2;
  float2 v[P];
};
template <typename T, int V>
__device__ __forceinline__ Lanes<V> lanes(const Chunk<T, V>& c) {
  Lanes<V> r;
#pragma unroll
  for (int i = 0; i < Lanes<V>::P; ++i)
    r.v[i] = make_float2(to_f(c.v[2 * i]), V == 1 ? 0.f : to_f(c.v[V == 1 ? 0 : 2 * i + 1]));
  return r;
}
template <typename T, int V>
__device__ __forceinline__ Chunk<T, V> chunk(const Lanes<V>& l) {
  Chunk<T, V> c;
#pragma unroll
  for (int i = 0; i < V; ++i) c.v[i] = from_f<T>(i % 2 ? l.v[i / 2].y : l.v[i / 2].x);
  return c;
}
template <int V>
__device__ __forceinline__ void set_lane(Lanes<V>& l, int i, float v) { (i % 2 ? l.v[i / 2].y : l.v[i / 2].x) = v; }
// The weights of V channels are V W neighbouring elements.
template <typename P, int V, int W>
__device__ __forceinline__ void load_weights_as(const P* w, const P* b, int c, Lanes<V> (&out)[W], Lanes<V>& bias) {
  constexpr int Q = V % 4 == 0 ? 4 : V % 2 == 0 ? 2 : 1;
#pragma unroll
  for (int q = 0; q < V * W / Q; ++q) {
    const Chunk<P, Q> k = load_whole<P, Q>(w + int64_t(c) * W + q * Q, true);
#pragma unroll
    for (int i = 0; i < Q; ++i) set_lane<V>(out[(q * Q + i) % W], (q * Q + i) / W, to_f(k.v[i]));
  }
#pragma unroll
  for (int q = 0; q < V / Q; ++q) {
    const Chunk<P, Q> k = load_whole<P, Q>(b + c + q * Q, b != nullptr);
#pragma unroll
    for (int i = 0; i < Q; ++i) set_lane<V>(bias, q * Q + i, to_f(k.v[i]));
  }
  if (V == 1) {  // the pair's other half
    bias.v[0].y = 0.f;
#pragma unroll
    for (int k = 0; k < W; ++k) out[k].v[0].y = 0.f;
  }
}
template <typename T, int V, int W>
__device__ __forceinline__ void load_weights(const ConvArgs& a, int c, Lanes<V> (&w)[W], Lanes<V>& bias) {
  if (a.wide)
    load_weights_as<float, V, W>(static_cast<const float*>(a.w), static_cast<const float*>(a.b), c, w, bias);
  else
    load_weights_as<T, V, W>(static_cast<const T*>(a.w), static_cast<const T*>(a.b), c, w, bias);
}

constexpr int kMarchThreads = 128;

// grid: (channel vectors / threads, pieces, batch).  V divides the channels.
template <typename T, int V, int W>
__global__ void __launch_bounds__(kMarchThreads, 6) conv_march_kernel(const ConvArgs a) {
  constexpr int P = Lanes<V>::P;
  const int c = (blockIdx.x * kMarchThreads + threadIdx.x) * V;
  if (c >= a.channels) return;
  const int64_t b = blockIdx.z;
  const int64_t len = live_length(a.lengths, a.length, b);
  const int64_t t0 = int64_t(blockIdx.y) * a.piece, t1 = min(t0 + a.piece, a.length), live = min(len, t1);
  const T* x = static_cast<const T*>(a.x) + b * a.xb + c;
  T* y = static_cast<T*>(a.y) + b * a.yb + c;
  constexpr int U = 4;  // positions per turn; those of the next turn are on their way meanwhile
  Chunk<T, V> next[U];
#pragma unroll
  for (int u = 0; u < U; ++u) next[u] = load_whole<T, V>(x + (t0 + u) * a.xs, t0 + u < live);
  Lanes<V> w[W], bias, win[W - 1 + U];
  load_weights<T, V, W>(a, c, w, bias);
#pragma unroll
  for (int k = 0; k < W - 1; ++k)
    win[k] = lanes<T, V>(t0 < len ? input_at<T, V, W>(a, b, t0 - (W - 1) + k, c) : Chunk<T, V>{});
  // `whole`: no position of the turn lies behind the sequence or the piece.
  auto turn = [&](auto whole, int64_t t) {
    constexpr bool WHOLE = decltype(whole)::value;
#pragma unroll
    for (int u = 0; u < U; ++u) win[W - 1 + u] = lanes<T, V>(next[u]);
#pragma unroll
    for (int u = 0; u < U; ++u) next[u] = load_whole<T, V>(x + (t + U + u) * a.xs, t + U + u < live);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      Lanes<V> p = bias;
#pragma unroll
      for (int i = 0; i < P; ++i) {
#pragma unroll
        for (int k = 0; k < W; ++k) p.v[i] = fma2(w[k].v[i], win[u + k].v[i], p.v[i]);
        if (a.silu) p.v[i] = mul2(p.v[i], sigmoid2(p.v[i]));
        if (!WHOLE && t + u >= len) p.v[i] = both(0.f);
      }
      store_whole<T, V>(y + (t + u) * a.ys, chunk<T, V>(p), WHOLE || t + u < t1);
    }
#pragma unroll
    for (int k = 0; k < W - 1; ++k) win[k] = win[U + k];
  };
  for (int64_t t = t0; t < t1; t += U) {
    if (t + U <= live) turn(std::true_type{}, t);
    else turn(std::false_type{}, t);
  }
  if (a.final_state && blockIdx.y == 0) {
    T* f = static_cast<T*>(a.final_state) + b * (W - 1) * a.channels + c;
#pragma unroll
    for (int k = 0; k < W - 1; ++k)
      store_whole<T, V>(f + int64_t(k) * a.channels, input_at<T, V, W>(a, b, len - (W - 1) + k, c), true);
  }
}

template <typename T, int V, int W>
__global__ void __launch_bounds__(kMarchThreads, 3) conv_march_backward_kernel(const ConvArgs a) {
  constexpr int P = Lanes<V>::P;
  const int c = (blockIdx.x * kMarchThreads + threadIdx.x) * V;
  if (c >= a.channels) return;
  const int64_t b = blockIdx.z;
  const int64_t len = live_length(a.lengths, a.length, b);
  const int64_t t0 = int64_t(blockIdx.y) * a.piece, t1 = min(t0 + a.piece, a.length);
  const int64_t last = min(len, t1 + W - 1);  // positions that this piece reads
  const T* x = static_cast<const T*>(a.x) + b * a.xb + c;
  const T* dy = static_cast<const T*>(a.dy) + b * a.dyb + c;
  T* dx = static_cast<T*>(a.dx) + b * a.dxb + c;
  const T* df = a.dfinal ? static_cast<const T*>(a.dfinal) + b * (W - 1) * a.channels + c : nullptr;
  constexpr int U = 4;
  Chunk<T, V> nx[U], nd[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    nx[u] = load_whole<T, V>(x + (t0 + u) * a.xs, t0 + u < last);
    nd[u] = load_whole<T, V>(dy + (t0 + u) * a.dys, t0 + u < last);
  }
  Lanes<V> w[W], bias, xw[W - 1 + U], qw[W - 1 + U], dw[W], db;
  load_weights<T, V, W>(a, c, w, bias);
#pragma unroll
  for (int i = 0; i < P; ++i) {
    db.v[i] = both(0.f);
#pragma unroll
    for (int k = 0; k < W; ++k) dw[k].v[i] = both(0.f);
#pragma unroll
    for (int k = 0; k < W - 1; ++k) qw[k].v[i] = both(0.f);
  }
#pragma unroll
  for (int k = 0; k < W - 1; ++k)
    xw[k] = lanes<T, V>(t0 < len ? input_at<T, V, W>(a, b, t0 - (W - 1) + k, c) : Chunk<T, V>{});
  // Step j brings q[j] in and completes dx[j - W + 1]; q is zero from `len` on.  `whole`: all positions of the turn
  // belong to this piece and none to an edge of the sequence.
  auto turn = [&](auto whole, int64_t j0) {
    constexpr bool WHOLE = decltype(whole)::value;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      xw[W - 1 + u] = lanes<T, V>(nx[u]);
      qw[W - 1 + u] = lanes<T, V>(nd[u]);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      nx[u] = load_whole<T, V>(x + (j0 + U + u) * a.xs, j0 + U + u < last);
      nd[u] = load_whole<T, V>(dy + (j0 + U + u) * a.dys, j0 + U + u < last);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t j = j0 + u, t = j - (W - 1);
      Lanes<V> g;
#pragma unroll
      for (int i = 0; i < P; ++i) {
        float2 q = qw[W - 1 + u].v[i];
        if (a.silu) {
          float2 p = bias.v[i];
#pragma unroll
          for (int k = 0; k < W; ++k) p = fma2(w[k].v[i], xw[u + k].v[i], p);
          const float2 s = sigmoid2(p);
          q = mul2(q, mul2(s, fma2(p, make_float2(1.f - s.x, 1.f - s.y), both(1.f))));
          if (!WHOLE && j >= last) q = both(0.f);
          qw[W - 1 + u].v[i] = q;
        }
        const float2 own = WHOLE || j < t1 ? q : both(0.f);  // the others count towards dw in the next piece
        db.v[i] = add2(db.v[i], own);
#pragma unroll
        for (int k = 0; k < W; ++k) {
          dw[k].v[i] = fma2(own, xw[u + k].v[i], dw[k].v[i]);
          g.v[i] = k == 0 ? mul2(w[k].v[i], qw[W - 1 + u].v[i]) : fma2(w[k].v[i], qw[W - 1 + u - k].v[i], g.v[i]);
        }
      }
      if constexpr (WHOLE) {
        store_whole<T, V>(dx + t * a.dxs, chunk<T, V>(g), true);
      } else {
        // The first piece also completes the gradients of the W - 1 inputs before position 0.
        const bool edge = t < 0 && a.dinit && j < t1 + W - 1;
        if (df && t < len && t >= len - (W - 1) && (t >= t0 || edge)) {
          const Lanes<V> f = lanes<T, V>(load_whole<T, V>(df + (t - (len - (W - 1))) * a.channels, true));
#pragma unroll
          for (int i = 0; i < P; ++i) g.v[i] = add2(g.v[i], f.v[i]);
        }
#pragma unroll
        for (int i = 0; i < P; ++i)
          if (t >= len) g.v[i] = both(0.f);
        store_whole<T, V>(dx + t * a.dxs, chunk<T, V>(g), t >= t0 && t < t1);
        if (edge)
          store_whole<T, V>(static_cast<T*>(a.dinit) + (b * (W - 1) + t + W - 1) * a.channels + c, chunk<T, V>(g),
                            true);
      }
    }
#pragma unroll
    for (int k = 0; k < W - 1; ++k) {
      xw[k] = xw[U + k];
      qw[k] = qw[U + k];
    }
  };
  for (int64_t j0 = t0; j0 < t1 + W - 1; j0 += U) {
    // dx[t] of the turn: t0 <= t, and none of the last W - 1 positions, which the final state's gradient may join
    if (j0 >= t0 + W - 1 && j0 + U <= t1 && j0 + U <= len) turn(std::true_type{}, j0);
    else turn(std::false_type{}, j0);
  }
  float* part = a.part + (b * a.pieces + blockIdx.y) * (W + 1) * a.channels + c;
#pragma unroll
  for (int k = 0; k <= W; ++k)
    store_whole<float, V>(part + int64_t(k) * a.channels, chunk<float, V>(k < W ? dw[k < W ? k : 0] : db), true);
}

// ---- sequence contiguous ---------------------------------------------------------------
template <typename T>
__device__ __forceinline__ float line_input(const ConvArgs& a, const T* x, int64_t b, int c, int64_t t, int width) {
  if (t >= 0) return to_f(x[t]);
  if (!a.init) return 0.f;
  return to_f(static_cast<const T*>(a.init)[(b * (width - 1) + t + width - 1) * a.channels + c]);
}

// grid: (channels, pieces, batch)
template <typename T, int W>
__global__ void __launch_bounds__(256) conv_lines_kernel(const ConvArgs a) {
  const int c = blockIdx.x;
  const int64_t b = blockIdx.z, len = live_length(a.lengths, a.length, b);
  const int64_t t0 = int64_t(blockIdx.y) * a.piece, t1 = min(t0 + a.piece, a.length);
  const T* x = static_cast<const T*>(a.x) + b * a.xb + c * a.xs;
  T* y = static_cast<T*>(a.y) + b * a.yb + c * a.ys;
  float w[W];
#pragma unroll
  for (int k = 0; k < W; ++k) w[k] = conv_param<T>(a.w, a.wide, int64_t(c) * W + k);
  const float bias = a.b ? conv_param<T>(a.b, a.wide, c) : 0.f;
  for (int64_t t = t0 + threadIdx.x; t < t1; t += 256) {
    float p = bias;
    if (t < len) {
#pragma unroll
      for (int k = 0; k < W; ++k) p = fmaf(w[k], line_input<T>(a, x, b, c, t - (W - 1) + k, W), p);
      if (a.silu) p *= sigmoid(p);
    } else {
      p = 0.f;
    }
    y[t] = from_f<T>(p);
  }
  if (W > 1 && a.final_state && blockIdx.y == 0 && int(threadIdx.x) < W - 1) {
    const int64_t t = len - (W - 1) + threadIdx.x;
    static_cast<T*>(a.final_state)[(b * (W - 1) + threadIdx.x) * a.channels + c] =
        from_f<T>(line_input<T>(a, x, b, c, t, W));
  }
}

template <typename T, int W>
__global__ void __launch_bounds__(256) conv_lines_backward_kernel(const ConvArgs a) {
  __shared__ float sums[8][W + 1];
  const int c = blockIdx.x;
  const int64_t b = blockIdx.z, len = live_length(a.lengths, a.length, b);
  const int64_t t0 = int64_t(blockIdx.y) * a.piece, t1 = min(t0 + a.piece, a.length);
  const T* x = static_cast<const T*>(a.x) + b * a.xb + c * a.xs;
  const T* dy = static_cast<const T*>(a.dy) + b * a.dyb + c * a.dys;
  T* dx = static_cast<T*>(a.dx) + b * a.dxb + c * a.dxs;
  float w[W], dw[W + 1];
#pragma unroll
  for (int k = 0; k < W; ++k) w[k] = conv_param<T>(a.w, a.wide, int64_t(c) * W + k);
#pragma unroll
  for (int k = 0; k <= W; ++k) dw[k] = 0.f;
  const float bias = a.b ? conv_param<T>(a.b, a.wide, c) : 0.f;
  // The first piece starts W - 1 positions early: those are the initial state's.
  const int64_t lo = t0 == 0 && a.dinit ? 1 - W : t0;
  for (int64_t t = lo + threadIdx.x; t < t1; t += 256) {
    float g = 0.f;
    // q[t], .., q[t + W - 1] from the inputs t - W + 1, .., t + W - 1.
    float xin[2 * W - 1];
#pragma unroll
    for (int k = 0; k < 2 * W - 1; ++k) {
      const int64_t s = t - (W - 1) + k;
      xin[k] = s < len && s >= 1 - W ? line_input<T>(a, x, b, c, s, W) : 0.f;
    }
#pragma unroll
    for (int m = 0; m < W; ++m) {
      const int64_t s = t + m;
      float q = s >= 0 && s < len ? to_f(dy[s]) : 0.f;
      if (a.silu) {
        float p = bias;
#pragma unroll
        for (int k = 0; k < W; ++k) p = fmaf(w[k], xin[m + k], p);
        q = s >= 0 && s < len ? q * silu_slope(p) : 0.f;
      }
      g = fmaf(w[W - 1 - m], q, g);
      if (m == 0) {
#pragma unroll
        for (int k = 0; k < W; ++k) dw[k] = fmaf(q, xin[k], dw[k]);
        dw[W] += q;
      }
    }
    if (a.dfinal && t < len && t >= len - (W - 1))
      g += to_f(static_cast<const T*>(a.dfinal)[(b * (W - 1) + t - (len - (W - 1))) * a.channels + c]);
    g = t < len ? g : 0.f;
    if (t >= 0) dx[t] = from_f<T>(g);
    else static_cast<T*>(a.dinit)[(b * (W - 1) + t + W - 1) * a.channels + c] = from_f<T>(g);
  }
#pragma unroll
  for (int k = 0; k <= W; ++k) {
    const float s = warp_sum(dw[k]);
    if (threadIdx.x % 32 == 0) sums[threadIdx.x / 32][k] = s;
  }
  __syncthreads();
  if (threadIdx.x <= W) {
    float s = 0.f;
    for (int i = 0; i < 8; ++i) s += sums[i][threadIdx.x];
    a.part[((b * a.pieces + blockIdx.y) * (W + 1) + threadIdx.x) * a.channels + c] = s;
  }
}

// dw [channels, width] and dbias from `rows` partial rows of (width + 1) * channels values.
template <typename P>
__global__ void __launch_bounds__(1024) conv_params_kernel(const float* part, int64_t rows, int width, int channels,
                                                           P* dw, P* db) {
  __shared__ float sums[32][33];
  const int c = threadIdx.x % 32, r = threadIdx.x / 32;
  const int64_t n = int64_t(width + 1) * channels, i = int64_t(blockIdx.x) * 32 + c;
  float s = 0.f;
  if (i < n) {
    int64_t k = r;
    for (; k + 7 * 32 < rows; k += 8 * 32) {  // loads in flight together, added in order
      float v[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = part[(k + j * 32) * n + i];
#pragma unroll
      for (int j = 0; j < 8; ++j) s += v[j];
    }
    for (; k < rows; k += 32) s += part[k * n + i];
  }
  sums[r][c] = s;
  __syncthreads();
  s = warp_sum(sums[c][r]);
  const int64_t o = int64_t(blockIdx.x) * 32 + r;
  if (c == 0 && o < n) {
    const int k = int(o / channels), ch = int(o % channels);
    if (k < width) dw[int64_t(ch) * width + k] = from_f<P>(s);
    else if (db) db[ch] = from_f<P>(s);
  }
}

// ---- single position ---------------------------------------------------------------------
// A thread owns V channels of one sequence and has read all it needs before it writes, so that
// out_state may be the state itself.
template <typename T, int V>
__global__ void __launch_bounds__(128) conv_step_kernel(const ConvArgs a, int width, int64_t state_b, int64_t out_b) {
  const int per = a.channels / V;  // V divides the channels
  const int64_t i = int64_t(blockIdx.x) * 128 + threadIdx.x;
  const int64_t b = i / per;
  if (b >= a.length) return;  // `length` holds the batch here
  const int c = int(i % per) * V;
  const T* state = static_cast<const T*>(a.init) + b * state_b + c;
  T* out = static_cast<T*>(a.final_state) + b * out_b + c;
  Chunk<T, V> rows[8];
#pragma unroll
  for (int k = 0; k < 7; ++k)
    if (k < width - 1) rows[k] = load_whole<T, V>(state + int64_t(k) * a.channels, true);
  const Chunk<T, V> x = load_whole<T, V>(static_cast<const T*>(a.x) + b * a.xb + c, true);
  float p[V];
#pragma unroll
  for (int j = 0; j < V; ++j) {
    p[j] = a.b ? conv_param<T>(a.b, a.wide, c + j) : 0.f;
#pragma unroll
    for (int k = 0; k < 7; ++k)
      if (k < width - 1) p[j] = fmaf(conv_param<T>(a.w, a.wide, int64_t(c + j) * width + k), to_f(rows[k].v[j]), p[j]);
    p[j] = fmaf(conv_param<T>(a.w, a.wide, int64_t(c + j) * width + width - 1), to_f(x.v[j]), p[j]);
  }
  Chunk<T, V> o;
#pragma unroll
  for (int j = 0; j < V; ++j) o.v[j] = from_f<T>(a.silu ? p[j] * sigmoid(p[j]) : p[j]);
  store_whole<T, V>(static_cast<T*>(a.y) + b * a.yb + c, o, true);
#pragma unroll
  for (int k = 1; k < 7; ++k)
    if (k < width - 1) store_whole<T, V>(out + int64_t(k - 1) * a.channels, rows[k], true);
  if (width > 1) store_whole<T, V>(out + int64_t(width - 2) * a.channels, x, true);
}

// ---- host ------------------------------------------------------------------------------
static int conv_check(const bst_conv_desc* d) {
  if (!d) return fail(BST_ERR_INVALID, "null description");
  if (!layer_dtype(d->dtype)) return fail(BST_ERR_UNSUPPORTED, "the convolution runs in float32, bfloat16 or float16");
  if (d->param_dtype != d->dtype && d->param_dtype != BST_F32)
    return fail(BST_ERR_UNSUPPORTED, "convolution weights must have the input's type or float32");
  if (d->width < 1 || d->width > 8) return fail(BST_ERR_UNSUPPORTED, "the convolution's width must be 1 to 8");
  if (d->batch < 0 || d->length < 0 || d->channels < 0) return fail(BST_ERR_INVALID, "negative extent");
  if (d->batch > 65535) return fail(BST_ERR_UNSUPPORTED, "more than 65535 sequences");
  if (d->channels > (int64_t(1) << 30) || d->length > (int64_t(1) << 30))
    return fail(BST_ERR_UNSUPPORTED, "more than 2^30 channels or positions");
  return BST_OK;
}

// Positions per piece.  Longer pieces re-read less and leave fewer partial sums; shorter ones give
// the GPU more threads: at least 16 positions, at most what leaves `want` threads per SM.
static int conv_piece(const bst_conv_desc* d, bool backward) {
  const int64_t least = (d->length + 65534) / 65535;  // the grid's limit on pieces
  if (d->lines) return int(std::max<int64_t>(1024, least));
  const int64_t threads = std::max<int64_t>(1, d->batch * ((d->channels + 3) / 4));
  const int64_t want = int64_t(sm_count()) * (backward ? 1536 : 2048);
  const int64_t pieces = std::max<int64_t>(1, (want + threads - 1) / threads);
  int64_t piece = (d->length + pieces - 1) / pieces;
  piece = std::max<int64_t>(16, (piece + 7) / 8 * 8);
  return int(std::max(piece, least));
}

static ConvArgs conv_args(const bst_conv_desc* d, bool backward) {
  ConvArgs a{};
  a.xb = d->x_batch, a.xs = d->x_step, a.yb = d->y_batch, a.ys = d->y_step;
  a.dyb = d->dy_batch, a.dys = d->dy_step, a.dxb = d->dx_batch, a.dxs = d->dx_step;
  a.length = d->length, a.channels = int(d->channels), a.silu = d->silu != 0;
  a.wide = d->param_dtype == BST_F32 && d->dtype != BST_F32;
  a.piece = conv_piece(d, backward);
  a.pieces = int((d->length + a.piece - 1) / a.piece);
  return a;
}

template <class F>
static int with_width(int width, F&& f) {
  switch (width) {
    case 1: return f(std::integral_constant<int, 1>{});
    case 2: return f(std::integral_constant<int, 2>{});
    case 3: return f(std::integral_constant<int, 3>{});
    case 4: return f(std::integral_constant<int, 4>{});
    case 5: return f(std::integral_constant<int, 5>{});
    case 6: return f(std::integral_constant<int, 6>{});
    case 7: return f(std::integral_constant<int, 7>{});
    default: return f(std::integral_constant<int, 8>{});
  }
}

// Channels per thread of the marching kernels: a vector where everything is aligned to 16 bytes and the window fits
// the registers (W <= 4), else single channels.  Four channels (8 bytes in 16-bit types): eight halve the warps that
// fit, and with them the bytes under way (1 x 8192 x 4096 in bf16: 53 us with eight).
template <int VW, class F>
static int with_vector(const ConvArgs& a, int width, F&& f) {
  if (a.vec && width <= 4) return f(std::integral_constant<int, VW>{});
  return f(std::integral_constant<int, 1>{});
}

}  // namespace bst

using namespace bst;

extern "C" {

int bst_causal_conv_forward(const bst_conv_desc* d, const void* x, const void* weight, const void* bias,
                            const void* initial, const int32_t* lengths, void* y, void* final_state, void* stream) {
  clear_error();
  if (int rc = conv_check(d)) return rc;
  if (d->batch == 0 || d->channels == 0) return BST_OK;
  if (!weight || (d->length > 0 && (!x || !y))) return fail(BST_ERR_INVALID, "null device pointer");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  ConvArgs a = conv_args(d, false);
  a.x = x, a.w = weight, a.b = bias, a.init = initial, a.y = y, a.final_state = final_state, a.lengths = lengths;
  const int64_t per = 16 / layer_elem_size(d->dtype);
  a.vec = !d->lines && aligned16(x) && aligned16(y) && aligned16(initial) && aligned16(final_state) &&
          aligned16(weight) && aligned16(bias) &&
          (d->channels | a.xb | a.xs | a.yb | a.ys) % per == 0;
  if (d->length == 0 && !final_state) return BST_OK;
  const unsigned pieces = unsigned(std::max(a.pieces, 1));  // no positions: one piece hands the state on
  return with_type(d->dtype, [&](auto t) {
    using T = decltype(t);
    return with_width(d->width, [&](auto w) {
      constexpr int W = decltype(w)::value;
      if (d->lines) {
        conv_lines_kernel<T, W><<<dim3(unsigned(d->channels), pieces, unsigned(d->batch)), 256, 0, st>>>(a);
        return launched("conv_lines_kernel launch");
      }
      return with_vector<4>(a, W, [&](auto v) {
        constexpr int V = W <= 4 ? decltype(v)::value : 1;
        const unsigned cols = unsigned((d->channels + 128 * V - 1) / (128 * V));
        conv_march_kernel<T, V, W><<<dim3(cols, pieces, unsigned(d->batch)), 128, 0, st>>>(a);
        return launched("conv_march_kernel launch");
      });
    });
  });
}

int bst_causal_conv_workspace(const bst_conv_desc* d, int64_t* bytes) {
  clear_error();
  if (int rc = conv_check(d)) return rc;
  if (!bytes) return fail(BST_ERR_INVALID, "null output");
  const ConvArgs a = conv_args(d, true);
  *bytes = d->batch * a.pieces * (d->width + 1) * d->channels * 4;
  return BST_OK;
}

int bst_causal_conv_backward(const bst_conv_desc* d, const void* x, const void* weight, const void* bias,
                             const void* initial, const int32_t* lengths, const void* dy, const void* dfinal,
                             void* dx, void* dweight, void* dbias, void* dinitial, void* workspace,
                             int64_t workspace_bytes, void* stream) {
  int64_t need = 0;
  if (int rc = bst_causal_conv_workspace(d, &need)) return rc;
  if (d->channels == 0) return BST_OK;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int64_t es = layer_elem_size(d->dtype), per = 16 / es, ps = layer_elem_size(d->param_dtype);
  if (!weight || !dweight) return fail(BST_ERR_INVALID, "null device pointer");
  if (d->batch == 0 || d->length == 0) {
    BST_CUDA(cudaMemsetAsync(dweight, 0, size_t(d->channels * d->width * ps), st));
    if (dbias) BST_CUDA(cudaMemsetAsync(dbias, 0, size_t(d->channels * ps), st));
    const size_t edge = size_t(d->batch * (d->width - 1) * d->channels * es);
    if (dinitial && edge && dfinal) BST_CUDA(cudaMemcpyAsync(dinitial, dfinal, edge, cudaMemcpyDeviceToDevice, st));
    else if (dinitial && edge) BST_CUDA(cudaMemsetAsync(dinitial, 0, edge, st));
    return BST_OK;
  }
  if (!x || !dy || !dx) return fail(BST_ERR_INVALID, "null device pointer");
  if (!workspace || workspace_bytes < need || !aligned16(workspace))
    return fail(BST_ERR_INVALID, "the workspace must hold " + std::to_string(need) + " bytes, aligned to 16");
  ConvArgs a = conv_args(d, true);
  a.x = x, a.w = weight, a.b = bias, a.init = initial, a.lengths = lengths, a.dy = dy, a.dfinal = dfinal;
  a.dx = dx, a.dinit = dinitial, a.part = static_cast<float*>(workspace);
  a.vec = !d->lines && aligned16(x) && aligned16(dy) && aligned16(dx) && aligned16(initial) && aligned16(dfinal) &&
          aligned16(weight) && aligned16(bias) &&
          aligned16(dinitial) && (d->channels | a.xb | a.xs | a.dyb | a.dys | a.dxb | a.dxs) % per == 0;
  int rc = with_type(d->dtype, [&](auto t) {
    using T = decltype(t);
    return with_width(d->width, [&](auto w) {
      constexpr int W = decltype(w)::value;
      const dim3 lines(unsigned(d->channels), unsigned(a.pieces), unsigned(d->batch));
      if (d->lines) {
        conv_lines_backward_kernel<T, W><<<lines, 256, 0, st>>>(a);
        return launched("conv_lines_backward_kernel launch");
      }
      return with_vector<4>(a, W, [&](auto v) {
        constexpr int V = W <= 4 ? decltype(v)::value : 1;
        const unsigned cols = unsigned((d->channels + 128 * V - 1) / (128 * V));
        conv_march_backward_kernel<T, V, W>
            <<<dim3(cols, unsigned(a.pieces), unsigned(d->batch)), 128, 0, st>>>(a);
        return launched("conv_march_backward_kernel launch");
      });
    });
  });
  if (rc) return rc;
  const int64_t n = int64_t(d->width + 1) * d->channels;
  return with_type(d->param_dtype, [&](auto t) {
    using P = decltype(t);
    conv_params_kernel<P><<<unsigned((n + 31) / 32), 1024, 0, st>>>(a.part, d->batch * a.pieces, d->width, a.channels,
                                                                    static_cast<P*>(dweight), static_cast<P*>(dbias));
    return launched("conv_params_kernel launch");
  });
}

int bst_causal_conv_step(const bst_conv_desc* d, const void* x, const void* state, int64_t state_batch,
                         const void* weight, const void* bias, void* y, void* out_state, int64_t out_state_batch,
                         void* stream) {
  clear_error();
  if (int rc = conv_check(d)) return rc;
  if (d->batch == 0 || d->channels == 0) return BST_OK;
  if (!x || !weight || !y || (d->width > 1 && (!state || !out_state)))
    return fail(BST_ERR_INVALID, "null device pointer");
  ConvArgs a{};
  a.x = x, a.w = weight, a.b = bias, a.init = state, a.y = y, a.final_state = out_state;
  a.xb = d->x_batch, a.yb = d->y_batch, a.length = d->batch, a.channels = int(d->channels), a.silu = d->silu != 0;
  a.wide = d->param_dtype == BST_F32 && d->dtype != BST_F32;
  const int64_t per = 16 / layer_elem_size(d->dtype);
  a.vec = aligned16(x) && aligned16(y) && aligned16(state) && aligned16(out_state) &&
          (d->channels | a.xb | a.yb | state_batch | out_state_batch) % per == 0;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return with_type(d->dtype, [&](auto t) {
    using T = decltype(t);
    auto go = [&](auto v) {
      constexpr int V = decltype(v)::value;
      const int64_t threads = d->batch * ((d->channels + V - 1) / V);
      conv_step_kernel<T, V><<<unsigned((threads + 127) / 128), 128, 0, st>>>(a, d->width, state_batch,
                                                                              out_state_batch);
      return launched("conv_step_kernel launch");
    };
    // Few vectors leave most of the GPU idle: then a thread takes one pair (or one) of the elements.
    if (a.vec && d->batch * d->channels / per >= int64_t(sm_count()) * 128)
      return go(std::integral_constant<int, 16 / int(sizeof(T))>{});
    if (a.vec) return go(std::integral_constant<int, 2>{});
    return go(std::integral_constant<int, 1>{});
  });
}

}  // extern "C"
