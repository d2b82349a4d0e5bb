// bst_scan_step.cu — selective scan, one position for every sequence (bst_scan_step).
//
//   h' = exp(d A) h + d u B,   y = (sum_n C h' + D u) silu(z)
// The state is read and written once in fp32 (8 bytes per entry) and dwarfs everything else, so HBM
// bounds it; with a few sequences the launch does (256 x 4096 x 16 in bf16: 33 us on B200 for 143 MB, 4.3 TB/s of
// a plain copy's 6.55; 2 x 1030 x 24 in fp32: 2.2 us).  L lanes share a channel, each with vectors of V
// states, and reduce y over themselves.  A thread has read its states before it writes them, so that
// out_state may be the state itself.  The new state is computed as the scan's forward kernel does it, bit for
// bit (the same decay, near 1 by its series: a sequence of tokens gathers its errors as a sequence of positions
// does).  The series took 4 us at 256 x 4096 x 16; the work on step size and gate done once per channel, not once
// per lane, gave them back.
#include <algorithm>

#include "bst_scan.cuh"

namespace bst {

struct StepArgs {
  const void *u, *delta, *z, *B, *C;
  const float *A, *D, *dbias, *state;
  void* y;
  float* out;
  int64_t ub, db, zb, yb, Bb, Bg, Cb, Cg, sb, sc, ob, oc;
  int64_t batch;
  int channels, per_group, states, softplus;
};

// Small blocks start and end at different times, so that loads and stores overlap more (and a ninth fits the registers):
// 33 us at 256 x 4096 x 16, with 256 threads 37.
constexpr int kStepThreads = 128;

template <typename T, int V>
__device__ __forceinline__ void load_floats(const T* p, float (&v)[V]) {
  const Chunk<T, V> c = *reinterpret_cast<const Chunk<T, V>*>(p);
#pragma unroll
  for (int i = 0; i < V; ++i) v[i] = to_f(c.v[i]);
}

// L lanes per channel, V states per access (states % V == 0), K = ceil(states / (L V)) accesses per lane, NB sequences
// per thread: what belongs to the channel (A, D, the step's bias) is read once for them, and their states are on
// their way together.
template <typename T, int L, int V, int K, int NB>
__global__ void __launch_bounds__(kStepThreads) scan_step_kernel(const StepArgs a) {
  const int i = int(blockIdx.x) * (kStepThreads / L) + int(threadIdx.x) / L, l = threadIdx.x % L;
  const bool in = i < a.channels;
  const int c = in ? i : 0, g = c / a.per_group;
  const int64_t b0 = int64_t(blockIdx.y) * NB;
  // What a sequence's lanes share (step size, gate, the sum's end) is one lane's work: lane l has OWN of the sequences.
  constexpr int OWN = NB > L ? NB / L : 1;
  const int own = NB == 1 ? 0 : l * OWN % NB;
  float hv[NB][K][V], Av[K][V], d[OWN], du[OWN], u[OWN], z[OWN];
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int n = (k * L + l) * V;
#pragma unroll
    for (int j = 0; j < NB; ++j)
      if (n < a.states && b0 + j < a.batch) load_floats<float, V>(a.state + (b0 + j) * a.sb + c * a.sc + n, hv[j][k]);
    if (n < a.states) load_floats<float, V>(a.A + int64_t(c) * a.states + n, Av[k]);
  }
  const float bias = a.dbias ? a.dbias[c] : 0.f, skip = a.D ? a.D[c] : 0.f;
#pragma unroll
  for (int i = 0; i < OWN; ++i) {
    const int64_t b = b0 + own + i < a.batch ? b0 + own + i : 0;
    d[i] = to_f(static_cast<const T*>(a.delta)[b * a.db + c]);
    u[i] = to_f(static_cast<const T*>(a.u)[b * a.ub + c]);
    z[i] = a.z ? to_f(static_cast<const T*>(a.z)[b * a.zb + c]) : 0.f;
  }
#pragma unroll
  for (int i = 0; i < OWN; ++i) {
    d[i] = a.softplus ? softplus(d[i] + bias) : d[i] + bias;
    du[i] = d[i] * u[i];
  }
  const int lane = threadIdx.x % 32;
  float y[NB];
#pragma unroll
  for (int j = 0; j < NB; ++j) y[j] = 0.f;
#pragma unroll
  for (int j = 0; j < NB; ++j) {
    if (b0 + j >= a.batch) break;
    const int64_t b = b0 + j;
    const float dj = NB == 1 ? d[0] : __shfl_sync(0xffffffffu, d[j % OWN], lane - l + j / OWN);
    const float duj = NB == 1 ? du[0] : __shfl_sync(0xffffffffu, du[j % OWN], lane - l + j / OWN);
    const T* B = static_cast<const T*>(a.B) + b * a.Bb + g * a.Bg;
    const T* C = static_cast<const T*>(a.C) + b * a.Cb + g * a.Cg;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int n = (k * L + l) * V;
      if (n < a.states) {
        float Bv[V], Cv[V];
        load_floats<T, V>(B + n, Bv);
        load_floats<T, V>(C + n, Cv);
        Chunk<float, V> o;
        float e[V + V % 2];  // in pairs
#pragma unroll
        for (int v = 0; v < V; v += 2) {
          const float2 a2 = make_float2(Av[k][v] * kLog2e, Av[k][V == 1 ? 0 : v + 1] * kLog2e);
          const float2 q = decay(both(dj), a2);
          e[v] = q.x, e[v + 1] = q.y;
        }
#pragma unroll
        for (int v = 0; v < V; ++v) {
          o.v[v] = fmaf(e[v], hv[j][k][v], duj * Bv[v]);
          y[j] = fmaf(o.v[v], Cv[v], y[j]);
        }
        if (in) *reinterpret_cast<Chunk<float, V>*>(a.out + b * a.ob + c * a.oc + n) = o;
      }
    }
  }
  constexpr int SPLIT = NB < L ? NB : L;  // lanes that end with sums of their own
#pragma unroll
  for (int m = L / 2; m >= SPLIT; m >>= 1)
#pragma unroll
    for (int j = 0; j < NB; ++j) y[j] += __shfl_xor_sync(0xffffffffu, y[j], m);
  reduce_scatter<NB, SPLIT, 1>(y, lane);
  if (!in || l >= SPLIT) return;
#pragma unroll
  for (int i = 0; i < OWN; ++i) {
    const int64_t b = b0 + own + i;
    float v = fmaf(skip, u[i], y[i]);
    if (a.z) v *= z[i] * sigmoid(z[i]);
    if (b < a.batch) static_cast<T*>(a.y)[b * a.yb + c] = from_f<T>(v);
  }
}

}  // namespace bst

using namespace bst;

extern "C" int bst_scan_step(const bst_scan_desc* d, const void* u, const void* delta, const float* A, const void* B,
                             const void* C, const float* D, const void* z, const float* delta_bias,
                             const float* state, int64_t state_batch, int64_t state_channel, void* y,
                             float* out_state, int64_t out_batch, int64_t out_channel, void* stream) {
  clear_error();
  if (int rc = scan_check(d)) return rc;
  if (d->batch == 0 || d->channels == 0) return BST_OK;
  if (!u || !delta || !A || !B || !C || !state || !y || !out_state) return fail(BST_ERR_INVALID, "null device pointer");
  StepArgs a{};
  a.u = u, a.delta = delta, a.z = z, a.B = B, a.C = C, a.A = A, a.D = D, a.dbias = delta_bias, a.state = state;
  a.y = y, a.out = out_state;
  a.ub = d->u_batch, a.db = d->delta_batch, a.zb = d->z_batch, a.yb = d->y_batch;
  a.Bb = d->B_batch, a.Bg = d->B_group, a.Cb = d->C_batch, a.Cg = d->C_group;
  a.sb = state_batch, a.sc = state_channel, a.ob = out_batch, a.oc = out_channel;
  a.batch = d->batch, a.channels = int(d->channels), a.per_group = int(d->channels / d->groups);
  a.states = int(d->states), a.softplus = d->softplus != 0;
  const bool vec = aligned16(A) && aligned16(B) && aligned16(C) && aligned16(state) && aligned16(out_state) &&
                   (d->states | a.Bb | a.Bg | a.Cb | a.Cg | a.sb | a.sc | a.ob | a.oc) % 4 == 0;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return with_type(d->dtype, [&](auto t) {
    using T = decltype(t);
    using std::integral_constant;
    // Four sequences per thread where that leaves two full turns of blocks (256 x 4096 x 16 in blocks of 256: 57 us
    // with one, 36 with four), one where threads are scarce.
    auto go = [&](auto lc, auto vc, auto kc) {
      constexpr int L = decltype(lc)::value, V = decltype(vc)::value, K = decltype(kc)::value;
      const int64_t cols = (d->channels * L + kStepThreads - 1) / kStepThreads;
      auto launch = [&](auto nb) {
        constexpr int NB = decltype(nb)::value;
        const int64_t turns = (d->batch + NB - 1) / NB;
        if (turns > 65535) return fail(BST_ERR_UNSUPPORTED, "the step takes up to 65535 sequences (more in large batches)");
        scan_step_kernel<T, L, V, K, NB><<<dim3(unsigned(cols), unsigned(turns)), kStepThreads, 0, st>>>(a);
        return launched("scan_step_kernel launch");
      };
      if constexpr (K <= 2)
        if (cols * ((d->batch + 3) / 4) >= int64_t(sm_count()) * 32) return launch(integral_constant<int, 4>{});
      return launch(integral_constant<int, 1>{});
    };
    integral_constant<int, 1> one;
    integral_constant<int, 2> two;
    integral_constant<int, 4> four;
    integral_constant<int, 8> eight;
    if (!vec) return go(eight, one, eight);
    if (d->states <= 8) return go(two, four, one);
    if (d->states <= 16) return go(four, four, one);
    if (d->states <= 32) return go(eight, four, one);
    return go(eight, four, two);
  });
}
