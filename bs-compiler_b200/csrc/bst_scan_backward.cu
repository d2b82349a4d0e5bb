// bst_scan_backward.cu — selective scan: backward pass (bst_scan_backward).
//
// With e_t = dy_t silu(z_t) (the gradient of s_t = sum_n C_t h_t + D u_t) and the adjoint
//   g_t[n] = C_t[n] e_t + a_{t+1}[n] g_{t+1}[n],      w_t[n] = g_t[n] a_t[n] h_{t-1}[n],
// the gradients are
//   dC_t = e_t h_t, dB_t = g_t d_t u_t (summed over the group's channels),  dA = sum_t d_t w_t,
//   du_t = d_t sum_n g_t B_t + D e_t,  dd_t = sum_n (A w_t + g_t B_t u_t),  ddelta_t = dd_t softplus'(.),
//   dz_t = dy_t s_t silu'(z_t),  dD = sum e_t u_t,  ddelta_bias = sum ddelta_t,  dinitial = a_1 g_1.
//
// The states are needed backwards and kept nowhere: the forward pass saved every 16th, and a block
// recomputes the 16 of a tile from it into registers, walking the tiles from the last to the first.
// Two exponentials for each (position, channel, state) bound it, and the sums over states and over
// channels that each step asks for: they go through reduce_scatter over the lanes, dB and dC then
// through shared memory over the block's warps and through a partial array over the channel tiles.
#include <algorithm>

#include "bst_scan.cuh"

namespace bst {

template <class Sh>
struct BackwardShared {
  float4 step[kScanTile][Sh::CT / 2];         // (d, d', d u, d' u') of a channel pair
  float2 e[kScanTile][Sh::CT / 2];
  float2 B[kScanTile][Sh::NP], C[kScanTile][Sh::NP];
  float sum_y[kScanTile][Sh::CT];             // sum_n C h
  float sum_g[kScanTile][Sh::CT], sum_w[kScanTile][Sh::CT];  // sum_n g B, sum_n A log2(e) w
  float bc[Sh::W][kScanTile][2 * Sh::NP];     // per warp: dB, dC summed over its channels
};

// Sums of v over the rows of the block that share a column, by the thread of row 0.
template <class Sh, int V, int PER_ROW>
__device__ void column_sums(float (&v)[V], float* buf) {
  __syncthreads();
#pragma unroll
  for (int j = 0; j < V; ++j) buf[threadIdx.x * V + j] = v[j];
  __syncthreads();
  if (threadIdx.x < PER_ROW)
    for (int r = 1; r < Sh::NT / PER_ROW; ++r)
#pragma unroll
      for (int j = 0; j < V; ++j) v[j] += buf[(threadIdx.x + r * PER_ROW) * V + j];
}

template <typename T, class Sh>
__global__ void __launch_bounds__(Sh::NT) scan_backward_kernel(const ScanArgs a) {
  constexpr int S = Sh::S, GS = Sh::GS, PW = Sh::PW, CT = Sh::CT, NP = Sh::NP, NT = Sh::NT, W = Sh::W;
  using Share = TileShare<T, Sh>;
  constexpr int V = Share::V, CNT = Share::CNT;
  constexpr int BC = (kScanTile * NP + NT - 1) / NT;
  extern __shared__ __align__(16) unsigned char raw_shared[];
  BackwardShared<Sh>& m = *reinterpret_cast<BackwardShared<Sh>*>(raw_shared);

  const ScanWhere at = scan_where(a);
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  const int sg = lane % GS, pair = warp * PW + lane / GS;
  const int c0 = at.ct * CT, left = a.per_group - c0;
  const int64_t cbase = int64_t(at.g) * a.per_group + c0;
  const int64_t len = scan_length(a, at.b);
  const int64_t first = int64_t(at.seg) * a.seg_tiles * kScanTile;
  const int64_t stop = min(first + int64_t(a.seg_tiles) * kScanTile, a.length);
  const int64_t live = max(min(stop, len), first);

  const int c_lane = 2 * pair;
  float2 carry[S], a2[S], dA[S];  // carry: a_{t+1} g_{t+1}
#pragma unroll
  for (int s = 0; s < S; ++s) {
    const int n = sg * S + s;
    carry[s] = a2[s] = dA[s] = make_float2(0.f, 0.f);
    if (n < a.states) {
      if (c_lane < left) a2[s].x = a.A[(cbase + c_lane) * a.states + n] * kLog2e;
      if (c_lane + 1 < left) a2[s].y = a.A[(cbase + c_lane + 1) * a.states + n] * kLog2e;
      if (a.dfinal) {
        const float* p = a.dfinal + (at.b * a.channels + cbase + c_lane) * a.states + n;
        if (c_lane < left) carry[s].x = p[0];
        if (c_lane + 1 < left) carry[s].y = p[a.states];
      }
    }
  }
  const int col = Share::col();
  float skip[V], bias[V], dD[V], dbias[V];
#pragma unroll
  for (int i = 0; i < V; ++i) {
    skip[i] = a.D && col + i < left ? a.D[cbase + col + i] : 0.f;
    bias[i] = a.dbias && col + i < left ? a.dbias[cbase + col + i] : 0.f;
    dD[i] = dbias[i] = 0.f;
  }
  const T* u = static_cast<const T*>(a.u) + at.b * a.ub + cbase + col;
  const T* dl = static_cast<const T*>(a.delta) + at.b * a.db + cbase + col;
  const T* z = static_cast<const T*>(a.z) + at.b * a.zb + cbase + col;
  const T* dy = static_cast<const T*>(a.dy) + at.b * a.dyb + cbase + col;
  const int64_t dense = at.b * a.length * a.channels + cbase + col;  // of the contiguous gradients
  T* du = static_cast<T*>(a.du) + dense;
  T* ddl = static_cast<T*>(a.ddelta) + dense;
  T* dz = static_cast<T*>(a.dz) + dense;
  const T* B = static_cast<const T*>(a.B) + at.b * a.Bb + at.g * a.Bg;
  const T* C = static_cast<const T*>(a.C) + at.b * a.Cb + at.g * a.Cg;
  float* part = a.part_bc + ((at.b * a.groups + at.g) * a.col_tiles + at.ct) * a.length * 2 * NP;

  // Positions behind the sequence's end.
  Chunk<T, V> zero;
#pragma unroll
  for (int j = 0; j < V; ++j) zero.v[j] = from_f<T>(0.f);
  for (int64_t t = (live + kScanTile - 1) / kScanTile * kScanTile + int(threadIdx.x) / Share::PER_ROW; t < stop;
       t += Share::ROWS) {
    store_chunk<T, V>(du + t * a.channels, zero, left - col, a.vec);
    store_chunk<T, V>(ddl + t * a.channels, zero, left - col, a.vec);
    if (a.dz) store_chunk<T, V>(dz + t * a.channels, zero, left - col, a.vec);
  }

  for (int64_t tile = (live - first + kScanTile - 1) / kScanTile - 1; tile >= 0; --tile) {
    const int64_t t0 = first + tile * kScanTile;
    Chunk<T, V> cu[CNT], cd[CNT], cz[CNT], cy[CNT];
#pragma unroll
    for (int i = 0; i < CNT; ++i) {
      const int r = Share::row(i);
      const int64_t t = t0 + r;
      const int n = t < live ? left - col : 0;
      cu[i] = load_chunk<T, V>(u + t * a.us, n, a.vec);
      cd[i] = load_chunk<T, V>(dl + t * a.ds, n, a.vec);
      cz[i] = load_chunk<T, V>(z + t * a.zs, a.z ? n : 0, a.vec);
      cy[i] = load_chunk<T, V>(dy + t * a.dys, n, a.vec);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float raw = to_f(cd[i].v[j]) + bias[j];
        const float d = j < n ? (a.softplus ? softplus(raw) : raw) : 0.f;
        float* cell = reinterpret_cast<float*>(&m.step[r][(col + j) / 2]) + (col + j) % 2;
        cell[0] = d;
        cell[2] = d * to_f(cu[i].v[j]);
        float e = to_f(cy[i].v[j]);
        if (a.z) {
          const float zf = to_f(cz[i].v[j]);
          e *= zf * sigmoid(zf);
        }
        reinterpret_cast<float*>(&m.e[r][0])[col + j] = e;
      }
    }
#pragma unroll
    for (int i = 0; i < BC; ++i) {
      const int k = threadIdx.x + i * NT, r = k / NP, n = k % NP;
      if (r < kScanTile) {
        const bool on = t0 + r < live && n < a.states;
        const float vb = on ? to_f(B[(t0 + r) * a.Bs + n]) : 0.f, vc = on ? to_f(C[(t0 + r) * a.Cs + n]) : 0.f;
        m.B[r][n] = make_float2(vb, vb);
        m.C[r][n] = make_float2(vc, vc);
      }
    }
    float2 h0[S], h[kScanTile][S];
    {
      const float* k = a.saved + ((at.b * ((a.length + kScanTile - 1) / kScanTile) + t0 / kScanTile) * a.channels +
                                  cbase + c_lane) * NP + sg * S;
#pragma unroll
      for (int s = 0; s < S; ++s)
        h0[s] = make_float2(c_lane < left ? k[s] : 0.f, c_lane + 1 < left ? k[NP + s] : 0.f);
    }
    __syncthreads();

    // The tile's states, and sum_n C h for the gate's gradient.
    constexpr int UY = GS >= 2 ? GS / 2 : 1;
#pragma unroll
    for (int r0 = 0; r0 < kScanTile; r0 += UY) {
      float v[2 * UY];
#pragma unroll
      for (int j = 0; j < UY; ++j) {
        const int r = r0 + j;
        const float4 st = m.step[r][pair];
        float2 acc = make_float2(0.f, 0.f);
#pragma unroll
        for (int s = 0; s < S; ++s) {
          const float2 before = r == 0 ? h0[s] : h[r > 0 ? r - 1 : 0][s];
          const float2 x = decay(make_float2(st.x, st.y), a2[s]);
          h[r][s] = fma2(x, before, mul2(make_float2(st.z, st.w), m.B[r][sg * S + s]));
          acc = fma2(h[r][s], m.C[r][sg * S + s], acc);
        }
        v[2 * j] = acc.x;
        v[2 * j + 1] = acc.y;
      }
      if (a.z) {
        reduce_scatter<2 * UY, GS, 1>(v, lane);
        m.sum_y[r0 + sg / 2][c_lane + sg % 2] = v[0];
      }
    }

    // Backwards.  UG steps share the sums over states (4 values a step), UB those over channels.
    constexpr int UG = GS >= 4 ? GS / 4 : 1, NG = 4 * UG / GS;
    constexpr int UB = 2 * S >= PW ? 1 : PW / (2 * S), NB = 2 * S * UB / PW;
    constexpr int UU = UG > UB ? UG : UB;
#pragma unroll
    for (int r0 = kScanTile - UU; r0 >= 0; r0 -= UU) {
      float vg[UU][4], vb[UU][2 * S];
#pragma unroll
      for (int j = UU - 1; j >= 0; --j) {
        const int r = r0 + j;
        const float4 st = m.step[r][pair];
        const float2 d = make_float2(st.x, st.y), du2 = make_float2(st.z, st.w), e = m.e[r][pair];
        float2 sg2 = make_float2(0.f, 0.f), sw2 = make_float2(0.f, 0.f);
#pragma unroll
        for (int s = 0; s < S; ++s) {
          const float2 Bn = m.B[r][sg * S + s], Cn = m.C[r][sg * S + s];
          const float2 x = decay(d, a2[s]);
          const float2 before = r == 0 ? h0[s] : h[r > 0 ? r - 1 : 0][s];
          const float2 g = fma2(Cn, e, carry[s]);
          const float2 w = mul2(g, mul2(x, before));
          sw2 = fma2(w, a2[s], sw2);
          dA[s] = fma2(w, d, dA[s]);
          sg2 = fma2(g, Bn, sg2);
          const float2 pb = mul2(g, du2), pc = mul2(e, h[r][s]);
          vb[j][2 * s] = pb.x + pb.y;
          vb[j][2 * s + 1] = pc.x + pc.y;
          carry[s] = mul2(x, g);
        }
        vg[j][0] = sg2.x;
        vg[j][1] = sg2.y;
        vg[j][2] = sw2.x;
        vg[j][3] = sw2.y;
      }
#pragma unroll
      for (int q = 0; q < UU / UG; ++q) {
        float v[4 * UG];
#pragma unroll
        for (int i = 0; i < 4 * UG; ++i) v[i] = vg[q * UG + i / 4][i % 4];
        reduce_scatter<4 * UG, GS, 1>(v, lane);
#pragma unroll
        for (int i = 0; i < NG; ++i) {
          const int id = sg * NG + i, r = r0 + q * UG + id / 4, k = id % 4;
          (k < 2 ? m.sum_g : m.sum_w)[r][c_lane + k % 2] = v[i];
        }
      }
#pragma unroll
      for (int q = 0; q < UU / UB; ++q) {
        float v[2 * S * UB];
#pragma unroll
        for (int i = 0; i < 2 * S * UB; ++i) v[i] = vb[q * UB + i / (2 * S)][i % (2 * S)];
        reduce_scatter<2 * S * UB, PW, GS>(v, lane);
#pragma unroll
        for (int i = 0; i < NB; ++i) {
          const int id = lane / GS * NB + i, r = r0 + q * UB + id / (2 * S), k = id % (2 * S);
          m.bc[warp][r][(k % 2) * NP + sg * S + k / 2] = v[i];
        }
      }
    }
    __syncthreads();

#pragma unroll
    for (int i = 0; i < CNT; ++i) {
      const int r = Share::row(i);
      const int64_t t = t0 + r;
      if (t >= stop) continue;
      Chunk<T, V> ou, od, oz;
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float uf = to_f(cu[i].v[j]), yf = to_f(cy[i].v[j]);
        const float e = reinterpret_cast<const float*>(&m.e[r][0])[col + j];
        const float d = (reinterpret_cast<const float*>(&m.step[r][(col + j) / 2]) + (col + j) % 2)[0];
        const float gB = m.sum_g[r][col + j];
        float dd = fmaf(m.sum_w[r][col + j], kLn2, gB * uf);
        if (a.softplus) dd *= sigmoid(to_f(cd[i].v[j]) + bias[j]);
        if (t >= live) dd = 0.f;
        ou.v[j] = from_f<T>(fmaf(d, gB, skip[j] * e));
        od.v[j] = from_f<T>(dd);
        dD[j] = fmaf(e, uf, dD[j]);
        dbias[j] += dd;
        float gz = 0.f;
        if (a.z) {
          const float zf = to_f(cz[i].v[j]), s = sigmoid(zf);
          gz = yf * fmaf(skip[j], uf, m.sum_y[r][col + j]) * (s * fmaf(zf, 1.f - s, 1.f));
        }
        oz.v[j] = from_f<T>(gz);
      }
      store_chunk<T, V>(du + t * a.channels, ou, left - col, a.vec);
      store_chunk<T, V>(ddl + t * a.channels, od, left - col, a.vec);
      if (a.dz) store_chunk<T, V>(dz + t * a.channels, oz, left - col, a.vec);
    }
    for (int k = threadIdx.x; k < kScanTile * 2 * NP; k += NT) {
      const int r = k / (2 * NP), n = k % (2 * NP);
      float v = 0.f;
#pragma unroll
      for (int i = 0; i < W; ++i) v += m.bc[i][r][n];
      if (t0 + r < live) part[(t0 + r) * 2 * NP + n] = v;
    }
    __syncthreads();
  }

  if (a.dinit && at.seg == 0) {
#pragma unroll
    for (int s = 0; s < S; ++s) {
      const int n = sg * S + s;
      if (n < a.states) {
        float* p = a.dinit + (at.b * a.channels + cbase + c_lane) * a.states + n;
        if (c_lane < left) p[0] = carry[s].x;
        if (c_lane + 1 < left) p[a.states] = carry[s].y;
      }
    }
  }
  const int64_t prow = (at.b * a.segments + at.seg) * a.channels + cbase;
#pragma unroll
  for (int s = 0; s < S; ++s) {
    float* p = a.part_a + (prow + c_lane) * NP + sg * S + s;
    if (c_lane < left) p[0] = dA[s].x;
    if (c_lane + 1 < left) p[NP] = dA[s].y;
  }
  float* buf = &m.sum_y[0][0];  // sum_y, sum_g and sum_w: 48 CT floats for NT V = 16 CT / CNT
  column_sums<Sh, V, Share::PER_ROW>(dD, buf);
  column_sums<Sh, V, Share::PER_ROW>(dbias, buf);
  if (threadIdx.x < Share::PER_ROW)
#pragma unroll
    for (int j = 0; j < V; ++j)
      if (col + j < left) {
        a.part_d[(prow + col + j) * 2] = dD[j];
        a.part_d[(prow + col + j) * 2 + 1] = dbias[j];
      }
}

// dB, dC: sums of the channel tiles' partials, zero behind each sequence's end.
template <typename T>
__global__ void __launch_bounds__(256) scan_bc_kernel(const ScanArgs a, int np) {
  const int64_t i = int64_t(blockIdx.x) * 256 + threadIdx.x;
  const int n2 = int(i % (2 * np));
  int64_t r = i / (2 * np);
  const int64_t t = r % a.length;
  r /= a.length;
  const int g = int(r % a.groups);
  const int64_t b = r / a.groups;
  const int n = n2 % np;
  if (b >= a.batch || n >= a.states) return;
  float v = 0.f;
  if (t < scan_length(a, b)) {
    const float* p = a.part_bc + ((b * a.groups + g) * a.col_tiles * a.length + t) * 2 * np + n2;
    for (int k = 0; k < a.col_tiles; ++k) v += p[int64_t(k) * a.length * 2 * np];
  }
  T* out = static_cast<T*>(n2 < np ? a.dB : a.dC);
  out[((b * a.length + t) * a.groups + g) * a.states + n] = from_f<T>(v);
}

// dA, dD, ddelta_bias: sums over the sequences (and their segments).
__global__ void __launch_bounds__(256) scan_params_kernel(const ScanArgs a, int np, int rows, float* dA, float* dD,
                                                          float* dbias) {
  const int64_t i = int64_t(blockIdx.x) * 256 + threadIdx.x;
  const int n = int(i % (np + 2));
  const int64_t c = i / (np + 2);
  if (c >= a.channels) return;
  float v = 0.f;
  if (n < np) {
    if (n >= a.states) return;
    for (int k = 0; k < rows; ++k) v += a.part_a[(int64_t(k) * a.channels + c) * np + n];
    dA[c * a.states + n] = v;
  } else {
    for (int k = 0; k < rows; ++k) v += a.part_d[(int64_t(k) * a.channels + c) * 2 + n - np];
    float* out = n == np ? dD : dbias;
    if (out) out[c] = v;
  }
}

// ---- host ------------------------------------------------------------------------------
// The block shape for N states, as f(ScanShape).
template <class F>
static auto with_backward_shape(int64_t states, F&& f) {
  switch (scan_pad(states)) {
    case 4: return f(ScanShape<2, 2, 4>{});
    case 8: return f(ScanShape<2, 4, 4>{});
    case 16: return f(ScanShape<2, 8, 8>{});
    case 32: return f(ScanShape<2, 16, 8>{});
    default: return f(ScanShape<2, 32, 8>{});
  }
}

struct BackwardLayout {
  int64_t bc, pa, pd, total;  // byte offsets of part_bc (0), part_a, part_d
};
static BackwardLayout backward_layout(const bst_scan_desc* d, int segments) {
  const int64_t np = scan_pad(d->states);
  const int64_t ct = with_backward_shape(d->states, [](auto sh) { return int64_t(decltype(sh)::CT); });
  const int64_t per_group = d->channels / d->groups, tiles = (per_group + ct - 1) / ct;
  BackwardLayout l{};
  l.pa = d->batch * d->groups * tiles * d->length * 2 * np * 4;
  l.pd = l.pa + d->batch * segments * d->channels * np * 4;
  l.total = l.pd + d->batch * segments * d->channels * 2 * 4;
  return l;
}

int64_t scan_backward_workspace(const bst_scan_desc* d) { return backward_layout(d, 1).total; }

template <typename T, class Sh>
static int scan_backward_launch(ScanArgs a, cudaStream_t st) {
  a.col_tiles = (a.per_group + Sh::CT - 1) / Sh::CT;
  const int64_t blocks = int64_t(a.batch) * a.segments * a.groups * a.col_tiles;
  const int64_t outs = int64_t(a.batch) * a.length * a.groups * 2 * Sh::NP;
  if (blocks > INT_MAX || outs / 256 + 1 > INT_MAX)
    return fail(BST_ERR_UNSUPPORTED, "the scan's gradients need more than 2^31 blocks");
  constexpr int smem = int(sizeof(BackwardShared<Sh>));
  auto* kernel = scan_backward_kernel<T, Sh>;
  BST_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
  kernel<<<unsigned(blocks), Sh::NT, smem, st>>>(a);
  if (int rc = launched("scan_backward_kernel launch")) return rc;
  scan_bc_kernel<T><<<unsigned((outs + 255) / 256), 256, 0, st>>>(a, Sh::NP);
  return launched("scan_bc_kernel launch");
}

}  // namespace bst

using namespace bst;

extern "C" int bst_scan_backward(const bst_scan_desc* d, const void* u, const void* delta, const float* A,
                                 const void* B, const void* C, const float* D, const void* z, const float* delta_bias,
                                 const int32_t* lengths, const void* dy, const float* dfinal, const void* saved,
                                 void* du, void* ddelta, float* dA, void* dB, void* dC, float* dD, void* dz,
                                 float* ddelta_bias, float* dinitial, void* workspace, int64_t workspace_bytes,
                                 void* stream) {
  int64_t need = 0;
  if (int rc = bst_scan_workspace(d, BST_SCAN_BACKWARD, &need)) return rc;
  if (d->channels == 0) return BST_OK;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (!dA) return fail(BST_ERR_INVALID, "null device pointer");
  if (d->batch == 0 || d->length == 0) {
    BST_CUDA(cudaMemsetAsync(dA, 0, size_t(d->channels * d->states) * 4, st));
    if (dD) BST_CUDA(cudaMemsetAsync(dD, 0, size_t(d->channels) * 4, st));
    if (ddelta_bias) BST_CUDA(cudaMemsetAsync(ddelta_bias, 0, size_t(d->channels) * 4, st));
    const size_t n = size_t(d->batch * d->channels * d->states) * 4;
    if (dinitial && n && dfinal) BST_CUDA(cudaMemcpyAsync(dinitial, dfinal, n, cudaMemcpyDeviceToDevice, st));
    else if (dinitial && n) BST_CUDA(cudaMemsetAsync(dinitial, 0, n, st));
    return BST_OK;
  }
  if (!u || !delta || !A || !B || !C || !dy || !saved || !du || !ddelta || !dB || !dC || (z && !dz))
    return fail(BST_ERR_INVALID, "null device pointer");
  if (!workspace || workspace_bytes < need || !aligned16(workspace))
    return fail(BST_ERR_INVALID, "the workspace must hold " + std::to_string(need) + " bytes, aligned to 16");
  ScanArgs a = scan_args(d);
  a.u = u, a.delta = delta, a.A = A, a.B = B, a.C = C, a.D = D, a.z = z, a.dbias = delta_bias, a.lengths = lengths;
  a.dy = dy, a.dfinal = dfinal, a.saved = static_cast<float*>(const_cast<void*>(saved));
  a.du = du, a.ddelta = ddelta, a.dB = dB, a.dC = dC, a.dz = z ? dz : nullptr, a.dinit = dinitial;
  const BackwardLayout l = backward_layout(d, a.segments);
  char* ws = static_cast<char*>(workspace);
  a.part_bc = reinterpret_cast<float*>(ws);
  a.part_a = reinterpret_cast<float*>(ws + l.pa);
  a.part_d = reinterpret_cast<float*>(ws + l.pd);
  const int64_t per = 16 / layer_elem_size(d->dtype);
  a.vec = aligned16(u) && aligned16(delta) && aligned16(z) && aligned16(dy) && aligned16(du) && aligned16(ddelta) &&
          aligned16(dz) &&
          (a.per_group | a.ub | a.us | a.db | a.ds | (z ? a.zb | a.zs : 0) | a.dyb | a.dys) % per == 0;
  int rc = with_type(d->dtype, [&](auto t) {
    using T = decltype(t);
    return with_backward_shape(d->states, [&](auto sh) { return scan_backward_launch<T, decltype(sh)>(a, st); });
  });
  if (rc) return rc;
  const int np = scan_pad(d->states);
  const int64_t n = d->channels * (np + 2);
  scan_params_kernel<<<unsigned((n + 255) / 256), 256, 0, st>>>(a, np, a.batch * a.segments, dA, dD, ddelta_bias);
  return launched("scan_params_kernel launch");
}
