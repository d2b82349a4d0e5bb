// bst_scan.cu — selective scan: forward pass (bst_scan_forward) and workspace sizes.
#include <algorithm>
#include <cstdlib>

#include "bst_scan.cuh"

namespace bst {

// One block: CT channels of one sequence, its tiles in order.
template <typename T, class Sh>
__global__ void __launch_bounds__(Sh::NT) scan_forward_kernel(const ScanArgs a) {
  constexpr int S = Sh::S, CH = Sh::CH, GS = Sh::GS, CT = Sh::CT, NP = Sh::NP, NT = Sh::NT;
  using Share = TileShare<T, Sh>;
  using States = StateShare<T, Sh>;
  constexpr int V = Share::V, CNT = Share::CNT, VB = States::V;
  __shared__ Step<CH> s_step[kScanTile][CT / CH];
  __shared__ __align__(16) float s_B[kScanTile][NP], s_C[kScanTile][NP];
  __shared__ __align__(16) float s_y[kScanTile][CT];
  __shared__ Chunk<T, V> s_u[2][CNT][NT], s_dl[2][CNT][NT], s_z[2][CNT][NT];
  __shared__ Chunk<T, VB> s_rawB[2][States::CNT][NT], s_rawC[2][States::CNT][NT];

  const ScanWhere at = scan_where(a);
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  const int sg = lane % GS, cell = warp * (32 / GS) + lane / GS;
  const int c0 = at.ct * CT, left = a.per_group - c0;  // channels of the group from this tile on
  const int64_t cbase = int64_t(at.g) * a.per_group + c0;
  const int64_t len = scan_length(a, at.b);
  const int64_t first = int64_t(at.seg) * a.seg_tiles * kScanTile;
  const int64_t stop = min(first + int64_t(a.seg_tiles) * kScanTile, a.length);  // of this segment
  const int64_t live = min(stop, len);

  const int c_lane = CH * cell;
  Pairs<S> h[CH], a2[CH];
#pragma unroll
  for (int c = 0; c < CH; ++c)
#pragma unroll
    for (int s = 0; s < S; ++s) {
      const int n = sg * S + s;
      const bool on = n < a.states && c_lane + c < left;
      const int64_t i = (cbase + c_lane + c) * a.states + n;
      (s % 2 ? a2[c].v[s / 2].y : a2[c].v[s / 2].x) = on ? a.A[i] * kLog2e : 0.f;
      (s % 2 ? h[c].v[s / 2].y : h[c].v[s / 2].x) = on && a.init ? a.init[at.b * a.channels * a.states + i] : 0.f;
    }
  const int col = Share::col();
  float skip[V], bias[V];
#pragma unroll
  for (int i = 0; i < V; ++i) {
    skip[i] = a.D && col + i < left ? a.D[cbase + col + i] : 0.f;
    bias[i] = a.dbias && col + i < left ? a.dbias[cbase + col + i] : 0.f;
  }
  const T* u = static_cast<const T*>(a.u) + at.b * a.ub + cbase + col;
  const T* dl = static_cast<const T*>(a.delta) + at.b * a.db + cbase + col;
  const T* z = static_cast<const T*>(a.z) + at.b * a.zb + cbase + col;
  T* y = static_cast<T*>(a.y) + at.b * a.yb + cbase + col;
  const T* B = static_cast<const T*>(a.B) + at.b * a.Bb + at.g * a.Bg;
  const T* C = static_cast<const T*>(a.C) + at.b * a.Cb + at.g * a.Cg;

  // Two tiles are on their way while a third is worked on.
  auto fetch = [&](int64_t t0, int slot) {
#pragma unroll
    for (int i = 0; i < CNT; ++i) {
      const int64_t t = t0 + Share::row(i);
      const int n = t < live ? left - col : 0;
      stage_chunk<T, V>(&s_u[slot][i][threadIdx.x], u + t * a.us, static_cast<const T*>(a.u), n, a.mode_act);
      stage_chunk<T, V>(&s_dl[slot][i][threadIdx.x], dl + t * a.ds, static_cast<const T*>(a.delta), n, a.mode_act);
      if (a.z) stage_chunk<T, V>(&s_z[slot][i][threadIdx.x], z + t * a.zs, static_cast<const T*>(a.z), n, a.mode_act);
    }
#pragma unroll
    for (int i = 0; i < States::CNT; ++i) {
      const int k = States::item(i), n = States::state(k);
      const int64_t t = t0 + States::row(k);
      const int m = k < States::ITEMS && t < live ? a.states - n : 0;
      stage_chunk<T, VB>(&s_rawB[slot][i][threadIdx.x], B + t * a.Bs + n, B, m, a.mode_bc);
      stage_chunk<T, VB>(&s_rawC[slot][i][threadIdx.x], C + t * a.Cs + n, C, m, a.mode_bc);
    }
  };
  if (first < live) fetch(first, 0);
  copy_commit();
  if (first + kScanTile < live) fetch(first + kScanTile, 1);
  copy_commit();
  int slot = 0;
  for (int64_t t0 = first; t0 < live; t0 += kScanTile, slot ^= 1) {
    copy_wait<1>();
    Chunk<T, V> cu[CNT], cz[CNT];
#pragma unroll
    for (int i = 0; i < CNT; ++i) {
      const int r = Share::row(i);
      const int n = t0 + r < live ? left - col : 0;
      cu[i] = s_u[slot][i][threadIdx.x];
      cz[i] = s_z[slot][i][threadIdx.x];
      const Chunk<T, V> cd = s_dl[slot][i][threadIdx.x];
      float d[V], du[V];
#pragma unroll
      for (int j = 0; j < V; ++j) d[j] = to_f(cd.v[j]) + bias[j];
      if (a.softplus) by_two<V>(d, softplus, softplus2);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        d[j] = j < n ? d[j] : 0.f;
        du[j] = d[j] * to_f(cu[i].v[j]);
      }
      put_steps<CH, V>(s_step[r], col, d, du);
    }
#pragma unroll
    for (int i = 0; i < States::CNT; ++i) {
      const int k = States::item(i);
      if (k < States::ITEMS) {
        const Chunk<T, VB> cb = s_rawB[slot][i][threadIdx.x], cc = s_rawC[slot][i][threadIdx.x];
#pragma unroll
        for (int j = 0; j < VB; ++j) {
          s_B[States::row(k)][States::state(k) + j] = to_f(cb.v[j]);
          s_C[States::row(k)][States::state(k) + j] = to_f(cc.v[j]);
        }
      }
    }
    if (a.saved) {
      float* k = a.saved + ((at.b * ((a.length + kScanTile - 1) / kScanTile) + t0 / kScanTile) * a.channels + cbase +
                            c_lane) * NP + sg * S;
#pragma unroll
      for (int c = 0; c < CH; ++c)
        if (c_lane + c < left) *reinterpret_cast<Pairs<S>*>(k + c * NP) = h[c];
    }
    __syncthreads();
    if (t0 + 2 * kScanTile < live) fetch(t0 + 2 * kScanTile, slot);
    copy_commit();
    constexpr int U = GS > CH ? GS / CH : 1;  // steps whose sums over the states are joined together
    constexpr int OUT = U * CH / GS;          // of which each lane ends with so many
#pragma unroll
    for (int r0 = 0; r0 < kScanTile; r0 += U) {
      float v[U * CH];
#pragma unroll
      for (int j = 0; j < U; ++j) {
        const Step<CH> st = s_step[r0 + j][cell];
        const Pairs<S> Bn = *reinterpret_cast<const Pairs<S>*>(&s_B[r0 + j][sg * S]);
        const Pairs<S> Cn = *reinterpret_cast<const Pairs<S>*>(&s_C[r0 + j][sg * S]);
#pragma unroll
        for (int c = 0; c < CH; ++c) {
          float2 acc = make_float2(0.f, 0.f);
#pragma unroll
          for (int s = 0; s < S / 2; ++s) {
            const float2 e = decay(both(st.d[c]), a2[c].v[s]);
            h[c].v[s] = fma2(e, h[c].v[s], mul2(both(st.du[c]), Bn.v[s]));
            acc = s == 0 ? mul2(h[c].v[s], Cn.v[s]) : fma2(h[c].v[s], Cn.v[s], acc);
          }
          v[j * CH + c] = acc.x + acc.y;
        }
      }
      reduce_scatter<U * CH, GS, 1>(v, lane);
#pragma unroll
      for (int i = 0; i < OUT; ++i) {
        const int id = sg * OUT + i;
        s_y[r0 + id / CH][c_lane + id % CH] = v[i];
      }
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < CNT; ++i) {
      const int r = Share::row(i);
      const int64_t t = t0 + r;
      if (t >= stop) continue;
      float v[V], g[V];
#pragma unroll
      for (int j = 0; j < V; ++j) v[j] = fmaf(skip[j], to_f(cu[i].v[j]), s_y[r][col + j]);
      if (a.z) {
#pragma unroll
        for (int j = 0; j < V; ++j) g[j] = to_f(cz[i].v[j]);
        by_two<V>(g, [](float x) { return x * sigmoid(x); }, [](float2 x) { return mul2(x, sigmoid2(x)); });
#pragma unroll
        for (int j = 0; j < V; ++j) v[j] *= g[j];
      }
      Chunk<T, V> o;
#pragma unroll
      for (int j = 0; j < V; ++j) o.v[j] = from_f<T>(t < live ? v[j] : 0.f);
      store_chunk<T, V>(y + t * a.ys, o, left - col, a.vec);
    }
  }
  // Positions behind the sequence's end.
  const int64_t done = max(first, (live + kScanTile - 1) / kScanTile * kScanTile);
  Chunk<T, V> zero;
#pragma unroll
  for (int j = 0; j < V; ++j) zero.v[j] = from_f<T>(0.f);
  for (int64_t t = done + int(threadIdx.x) / Share::PER_ROW; t < stop; t += Share::ROWS)
    store_chunk<T, V>(y + t * a.ys, zero, left - col, a.vec);

  if (a.final_state && at.seg == a.segments - 1) {
#pragma unroll
    for (int c = 0; c < CH; ++c)
#pragma unroll
      for (int s = 0; s < S; ++s) {
        const int n = sg * S + s;
        if (n < a.states && c_lane + c < left)
          a.final_state[(at.b * a.channels + cbase + c_lane + c) * a.states + n] =
              s % 2 ? h[c].v[s / 2].y : h[c].v[s / 2].x;
      }
  }
}

// ---- host ------------------------------------------------------------------------------
int scan_check(const bst_scan_desc* d) {
  if (!d) return fail(BST_ERR_INVALID, "null description");
  if (!layer_dtype(d->dtype)) return fail(BST_ERR_UNSUPPORTED, "the scan runs in float32, bfloat16 or float16");
  if (d->batch < 0 || d->length < 0 || d->channels < 0) return fail(BST_ERR_INVALID, "negative extent");
  if (d->states < 1 || d->states > 64) return fail(BST_ERR_UNSUPPORTED, "the scan's states must be 1 to 64");
  if (d->groups < 1 || d->channels % d->groups) return fail(BST_ERR_INVALID, "groups must divide the channels");
  if (d->channels > (int64_t(1) << 24) || d->length > (int64_t(1) << 30) || d->batch > (int64_t(1) << 24))
    return fail(BST_ERR_UNSUPPORTED, "more than 2^24 channels or sequences, or 2^30 positions");
  return BST_OK;
}

ScanArgs scan_args(const bst_scan_desc* d) {
  ScanArgs a{};
  a.ub = d->u_batch, a.us = d->u_step, a.db = d->delta_batch, a.ds = d->delta_step;
  a.zb = d->z_batch, a.zs = d->z_step, a.yb = d->y_batch, a.ys = d->y_step, a.dyb = d->dy_batch, a.dys = d->dy_step;
  a.Bb = d->B_batch, a.Bs = d->B_step, a.Bg = d->B_group, a.Cb = d->C_batch, a.Cs = d->C_step, a.Cg = d->C_group;
  a.length = d->length, a.channels = int(d->channels), a.groups = int(d->groups);
  a.per_group = int(d->channels / d->groups), a.states = int(d->states), a.batch = int(d->batch);
  a.softplus = d->softplus != 0;
  a.segments = 1;
  a.seg_tiles = int((d->length + kScanTile - 1) / kScanTile);
  return a;
}

int64_t scan_saved_bytes(const bst_scan_desc* d) {
  return d->batch * ((d->length + kScanTile - 1) / kScanTile) * d->channels * scan_pad(d->states) * 4;
}

int64_t scan_backward_workspace(const bst_scan_desc* d);  // bst_scan_backward.cu

template <typename T, class Sh>
static int scan_forward_launch(ScanArgs a, cudaStream_t st) {
  a.col_tiles = (a.per_group + Sh::CT - 1) / Sh::CT;
  const int64_t blocks = int64_t(a.batch) * a.segments * a.groups * a.col_tiles;
  if (blocks > INT_MAX) return fail(BST_ERR_UNSUPPORTED, "the scan needs more than 2^31 blocks");
  scan_forward_kernel<T, Sh><<<unsigned(blocks), Sh::NT, 0, st>>>(a);
  return launched("scan_forward_kernel launch");
}

}  // namespace bst

using namespace bst;

extern "C" {

int bst_scan_workspace(const bst_scan_desc* d, int32_t what, int64_t* bytes) {
  clear_error();
  if (int rc = scan_check(d)) return rc;
  if (!bytes) return fail(BST_ERR_INVALID, "null output");
  if (what == BST_SCAN_FORWARD) *bytes = 0;
  else if (what == BST_SCAN_BACKWARD) *bytes = scan_backward_workspace(d);
  else if (what == BST_SCAN_SAVED) *bytes = scan_saved_bytes(d);
  else return fail(BST_ERR_INVALID, "unknown workspace");
  return BST_OK;
}

int bst_scan_forward(const bst_scan_desc* d, const void* u, const void* delta, const float* A, const void* B,
                     const void* C, const float* D, const void* z, const float* delta_bias, const float* initial,
                     const int32_t* lengths, void* y, float* final_state, void* saved, void* workspace,
                     int64_t workspace_bytes, void* stream) {
  int64_t need = 0;
  if (int rc = bst_scan_workspace(d, BST_SCAN_FORWARD, &need)) return rc;
  if (d->batch == 0 || d->channels == 0) return BST_OK;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (d->length == 0) {  // the state passes through
    if (!final_state) return BST_OK;
    const size_t n = size_t(d->batch * d->channels * d->states) * 4;
    if (initial) BST_CUDA(cudaMemcpyAsync(final_state, initial, n, cudaMemcpyDeviceToDevice, st));
    else BST_CUDA(cudaMemsetAsync(final_state, 0, n, st));
    return BST_OK;
  }
  if (!u || !delta || !A || !B || !C || !y) return fail(BST_ERR_INVALID, "null device pointer");
  if (need && (!workspace || workspace_bytes < need || !aligned16(workspace)))
    return fail(BST_ERR_INVALID, "the workspace must hold " + std::to_string(need) + " bytes, aligned to 16");
  ScanArgs a = scan_args(d);
  a.u = u, a.delta = delta, a.A = A, a.B = B, a.C = C, a.D = D, a.z = z, a.dbias = delta_bias, a.init = initial;
  a.lengths = lengths, a.y = y, a.final_state = final_state, a.saved = static_cast<float*>(saved);
  const int64_t per = 16 / layer_elem_size(d->dtype);
  a.vec = aligned16(u) && aligned16(delta) && aligned16(z) && aligned16(y) &&
          (a.per_group | a.ub | a.us | a.db | a.ds | (z ? a.zb | a.zs : 0) | a.yb | a.ys) % per == 0;
  const uint64_t es = uint64_t(layer_elem_size(d->dtype));
  auto at = [](const void* p) { return uint64_t(reinterpret_cast<uintptr_t>(p)); };
  a.mode_act = copy_mode(at(u) | at(delta) | at(z) | es * (a.per_group | a.ub | a.us | a.db | a.ds | (z ? a.zb | a.zs : 0)));
  a.mode_bc = copy_mode((at(B) | at(C) | es * (a.states | a.Bb | a.Bs | a.Bg | a.Cb | a.Cs | a.Cg)) % 4 ? 1 : 4);
  return with_type(d->dtype, [&](auto t) {
    using T = decltype(t);
    const int force = std::getenv("BST_S") ? std::atoi(std::getenv("BST_S")) : 2;
    switch (scan_pad(d->states)) {
      case 4: return scan_forward_launch<T, ScanShape<2, 2, 2, 2>>(a, st);
      case 8: return scan_forward_launch<T, ScanShape<4, 2, 2, 2>>(a, st);
      case 16:
        if (force == 1) return scan_forward_launch<T, ScanShape<2, 1, 8, 4>>(a, st);
        if (force == 2) return scan_forward_launch<T, ScanShape<4, 1, 4, 4>>(a, st);
        if (force == 3) return scan_forward_launch<T, ScanShape<2, 2, 8, 4>>(a, st);
        return scan_forward_launch<T, ScanShape<4, 2, 4, 4>>(a, st);
      case 32: return scan_forward_launch<T, ScanShape<4, 2, 8, 4>>(a, st);
      default: return scan_forward_launch<T, ScanShape<4, 2, 16, 4>>(a, st);
    }
  });
}

}  // extern "C"
