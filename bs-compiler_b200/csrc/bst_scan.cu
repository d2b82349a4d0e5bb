// bst_scan.cu — selective scan: forward pass (bst_scan_forward) and workspace sizes.
#include <algorithm>

#include "bst_scan.cuh"

namespace bst {

// One block: CT channels of one sequence, its tiles in order.
template <typename T, class Sh>
__global__ void __launch_bounds__(Sh::NT) scan_forward_kernel(const ScanArgs a) {
  constexpr int S = Sh::S, GS = Sh::GS, PW = Sh::PW, CT = Sh::CT, NP = Sh::NP, NT = Sh::NT;
  using Share = TileShare<T, Sh>;
  constexpr int V = Share::V, CNT = Share::CNT;
  constexpr int BC = kScanTile * NP / NT > 0 ? kScanTile * NP / NT : 1;  // elements of B (of C) per thread
  __shared__ float4 s_step[kScanTile][CT / 2];  // (d, d', d u, d' u') of a channel pair
  __shared__ float2 s_B[kScanTile][NP], s_C[kScanTile][NP];  // each value twice, as the paired operands want it
  __shared__ float s_y[kScanTile][CT];

  const ScanWhere at = scan_where(a);
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  const int sg = lane % GS, pair = warp * PW + lane / GS;
  const int c0 = at.ct * CT, left = a.per_group - c0;  // channels of the group from this tile on
  const int64_t cbase = int64_t(at.g) * a.per_group + c0;
  const int64_t len = scan_length(a, at.b);
  const int64_t first = int64_t(at.seg) * a.seg_tiles * kScanTile;
  const int64_t stop = min(first + int64_t(a.seg_tiles) * kScanTile, a.length);  // of this segment
  const int64_t live = min(stop, len);

  const int c_lane = 2 * pair;
  float2 h[S], a2[S];
#pragma unroll
  for (int s = 0; s < S; ++s) {
    const int n = sg * S + s;
    h[s] = a2[s] = make_float2(0.f, 0.f);
    if (n < a.states) {
      if (c_lane < left) a2[s].x = a.A[(cbase + c_lane) * a.states + n] * kLog2e;
      if (c_lane + 1 < left) a2[s].y = a.A[(cbase + c_lane + 1) * a.states + n] * kLog2e;
      if (a.init) {
        const float* p = a.init + (at.b * a.channels + cbase + c_lane) * a.states + n;
        if (c_lane < left) h[s].x = p[0];
        if (c_lane + 1 < left) h[s].y = p[a.states];
      }
    }
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

  for (int64_t t0 = first; t0 < live; t0 += kScanTile) {
    Chunk<T, V> cu[CNT], cz[CNT];
#pragma unroll
    for (int i = 0; i < CNT; ++i) {
      const int r = Share::row(i);
      const int64_t t = t0 + r;
      const int n = t < live ? left - col : 0;
      cu[i] = load_chunk<T, V>(u + t * a.us, n, a.vec);
      const Chunk<T, V> cd = load_chunk<T, V>(dl + t * a.ds, n, a.vec);
      cz[i] = load_chunk<T, V>(z + t * a.zs, a.z ? n : 0, a.vec);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float raw = to_f(cd.v[j]) + bias[j];
        const float d = j < n ? (a.softplus ? softplus(raw) : raw) : 0.f;
        float* cell = reinterpret_cast<float*>(&s_step[r][(col + j) / 2]) + (col + j) % 2;
        cell[0] = d;
        cell[2] = d * to_f(cu[i].v[j]);
      }
    }
#pragma unroll
    for (int i = 0; i < BC; ++i) {
      const int e = threadIdx.x + i * NT, r = e / NP, n = e % NP;
      if (r < kScanTile) {
        const bool on = t0 + r < live && n < a.states;
        const float vb = on ? to_f(B[(t0 + r) * a.Bs + n]) : 0.f, vc = on ? to_f(C[(t0 + r) * a.Cs + n]) : 0.f;
        s_B[r][n] = make_float2(vb, vb);
        s_C[r][n] = make_float2(vc, vc);
      }
    }
    if (a.saved) {
      float* k = a.saved + ((at.b * ((a.length + kScanTile - 1) / kScanTile) + t0 / kScanTile) * a.channels + cbase +
                            c_lane) * NP + sg * S;
#pragma unroll
      for (int s = 0; s < S; ++s) {
        if (c_lane < left) k[s] = h[s].x;
        if (c_lane + 1 < left) k[NP + s] = h[s].y;
      }
    }
    __syncthreads();
    constexpr int U = GS >= 2 ? GS / 2 : 1;  // steps whose sums are joined together
#pragma unroll 1
    for (int r0 = 0; r0 < kScanTile; r0 += U) {
      float v[2 * U];
#pragma unroll
      for (int j = 0; j < U; ++j) {
        const float4 st = s_step[r0 + j][pair];
        float2 acc = make_float2(0.f, 0.f);
#pragma unroll
        for (int s = 0; s < S; ++s) {
          const float2 e = decay(make_float2(st.x, st.y), a2[s]);
          h[s] = fma2(e, h[s], mul2(make_float2(st.z, st.w), s_B[r0 + j][sg * S + s]));
          acc = fma2(h[s], s_C[r0 + j][sg * S + s], acc);
        }
        v[2 * j] = acc.x;
        v[2 * j + 1] = acc.y;
      }
      if constexpr (GS == 1) {
        s_y[r0][c_lane] = v[0];
        s_y[r0][c_lane + 1] = v[1];
      } else {
        reduce_scatter<2 * U, GS, 1>(v, lane);
        s_y[r0 + sg / 2][c_lane + sg % 2] = v[0];
      }
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < CNT; ++i) {
      const int r = Share::row(i);
      const int64_t t = t0 + r;
      if (t >= stop) continue;
      Chunk<T, V> o;
#pragma unroll
      for (int j = 0; j < V; ++j) {
        float v = fmaf(skip[j], to_f(cu[i].v[j]), s_y[r][col + j]);
        if (a.z) {
          const float zf = to_f(cz[i].v[j]);
          v *= zf * sigmoid(zf);
        }
        o.v[j] = from_f<T>(t < live ? v : 0.f);
      }
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
    for (int s = 0; s < S; ++s) {
      const int n = sg * S + s;
      if (n < a.states) {
        float* p = a.final_state + (at.b * a.channels + cbase + c_lane) * a.states + n;
        if (c_lane < left) p[0] = h[s].x;
        if (c_lane + 1 < left) p[a.states] = h[s].y;
      }
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
  return with_type(d->dtype, [&](auto t) {
    using T = decltype(t);
    switch (scan_pad(d->states)) {
      case 4: return scan_forward_launch<T, ScanShape<2, 2, 4>>(a, st);
      case 8: return scan_forward_launch<T, ScanShape<4, 2, 4>>(a, st);
      case 16: return scan_forward_launch<T, ScanShape<4, 4, 4>>(a, st);
      case 32: return scan_forward_launch<T, ScanShape<4, 8, 4>>(a, st);
      default: return scan_forward_launch<T, ScanShape<4, 16, 4>>(a, st);
    }
  });
}

}  // extern "C"
