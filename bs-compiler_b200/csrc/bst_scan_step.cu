// bst_scan_step.cu — selective scan, one position for every sequence (bst_scan_step).
//
//   h' = exp(d A) h + d u B,   y = (sum_n C h' + D u) silu(z)
// The state is read and written once in fp32 (8 bytes per entry) and dwarfs everything else, so HBM
// bounds it; with a few sequences the launch does.  L lanes share a channel, each with vectors of V
// states, and reduce y over themselves; a thread has read its states before it writes them, so that
// out_state may be the state itself.
#include <algorithm>

#include "bst_scan.cuh"

namespace bst {

struct StepArgs {
  const void *u, *delta, *z, *B, *C;
  const float *A, *D, *dbias, *state;
  void* y;
  float* out;
  int64_t ub, db, zb, yb, Bb, Bg, Cb, Cg, sb, sc, ob, oc;
  int64_t rows;  // batch * channels
  int channels, per_group, states, softplus;
};

template <typename T, int V>
__device__ __forceinline__ void load_floats(const T* p, float (&v)[V]) {
  const Chunk<T, V> c = *reinterpret_cast<const Chunk<T, V>*>(p);
#pragma unroll
  for (int i = 0; i < V; ++i) v[i] = to_f(c.v[i]);
}

// L lanes per channel, V states per access (states % V == 0).
template <typename T, int L, int V>
__global__ void __launch_bounds__(256) scan_step_kernel(const StepArgs a) {
  const int64_t row = (int64_t(blockIdx.x) * 256 + threadIdx.x) / L;
  const int l = threadIdx.x % L;
  const bool on = row < a.rows;
  const int64_t b = on ? row / a.channels : 0;
  const int c = on ? int(row % a.channels) : 0, g = c / a.per_group;
  const float raw = to_f(static_cast<const T*>(a.delta)[b * a.db + c]) + (a.dbias ? a.dbias[c] : 0.f);
  const float u = to_f(static_cast<const T*>(a.u)[b * a.ub + c]);
  const float d = a.softplus ? softplus(raw) : raw;
  const float du = d * u, d2 = d * kLog2e;
  const float* A = a.A + int64_t(c) * a.states;
  const float* h = a.state + b * a.sb + c * a.sc;
  float* out = a.out + b * a.ob + c * a.oc;
  const T* B = static_cast<const T*>(a.B) + b * a.Bb + g * a.Bg;
  const T* C = static_cast<const T*>(a.C) + b * a.Cb + g * a.Cg;
  float y = 0.f;
  for (int n = l * V; n < a.states; n += L * V) {
    float hv[V], Av[V], Bv[V], Cv[V];
    load_floats<float, V>(h + n, hv);
    load_floats<float, V>(A + n, Av);
    load_floats<T, V>(B + n, Bv);
    load_floats<T, V>(C + n, Cv);
    Chunk<float, V> o;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      o.v[i] = fmaf(ex2(d2 * Av[i]), hv[i], du * Bv[i]);
      y = fmaf(o.v[i], Cv[i], y);
    }
    if (on) *reinterpret_cast<Chunk<float, V>*>(out + n) = o;
  }
#pragma unroll
  for (int m = L / 2; m >= 1; m >>= 1) y += __shfl_xor_sync(0xffffffffu, y, m);
  if (on && l == 0) {
    if (a.D) y = fmaf(a.D[c], u, y);
    if (a.z) {
      const float z = to_f(static_cast<const T*>(a.z)[b * a.zb + c]);
      y *= z * sigmoid(z);
    }
    static_cast<T*>(a.y)[b * a.yb + c] = from_f<T>(y);
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
  a.rows = d->batch * d->channels, a.channels = int(d->channels), a.per_group = int(d->channels / d->groups);
  a.states = int(d->states), a.softplus = d->softplus != 0;
  const bool vec = aligned16(A) && aligned16(B) && aligned16(C) && aligned16(state) && aligned16(out_state) &&
                   (d->states | a.Bb | a.Bg | a.Cb | a.Cg | a.sb | a.sc | a.ob | a.oc) % 4 == 0;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return with_type(d->dtype, [&](auto t) {
    using T = decltype(t);
    auto go = [&](auto lc, auto vc) {
      constexpr int L = decltype(lc)::value, V = decltype(vc)::value;
      const int64_t blocks = (a.rows * L + 255) / 256;
      if (blocks > INT_MAX) return fail(BST_ERR_UNSUPPORTED, "the step needs more than 2^31 blocks");
      scan_step_kernel<T, L, V><<<unsigned(blocks), 256, 0, st>>>(a);
      return launched("scan_step_kernel launch");
    };
    using std::integral_constant;
    if (!vec) return go(integral_constant<int, 8>{}, integral_constant<int, 1>{});
    if (d->states <= 8) return go(integral_constant<int, 2>{}, integral_constant<int, 4>{});
    if (d->states <= 16) return go(integral_constant<int, 4>{}, integral_constant<int, 4>{});
    return go(integral_constant<int, 8>{}, integral_constant<int, 4>{});
  });
}
