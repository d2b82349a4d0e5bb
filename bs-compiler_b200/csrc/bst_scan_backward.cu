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

template <typename T, class Sh>
struct BackwardShared {
  using Share = TileShare<T, Sh>;
  using States = StateShare<T, Sh>;
  Step<Sh::CH> step[kScanTile][Sh::CT / Sh::CH];
  alignas(16) float e[kScanTile][Sh::CT];
  alignas(16) float B[kScanTile][Sh::NP], C[kScanTile][Sh::NP];
  alignas(16) float sum_y[kScanTile][Sh::CT];                     // sum_n C h
  float sum_g[kScanTile][Sh::CT], sum_w[kScanTile][Sh::CT];       // sum_n g B, sum_n A log2(e) w
  float bc[Sh::W][kScanTile][2 * Sh::NP];                         // per warp: dB, dC summed over its channels
  Chunk<T, Share::V> raw[2][4][Share::CNT][Sh::NT];               // u, delta, z, dy as they come
  Chunk<T, States::V> raw_bc[2][2][States::CNT][Sh::NT];
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
  constexpr int S = Sh::S, CH = Sh::CH, GS = Sh::GS, CT = Sh::CT, NP = Sh::NP, NT = Sh::NT, W = Sh::W;
  constexpr int LC = 32 / GS;  // lanes of a warp that share a state group
  using Share = TileShare<T, Sh>;
  using States = StateShare<T, Sh>;
  constexpr int V = Share::V, CNT = Share::CNT, VB = States::V;
  extern __shared__ __align__(16) unsigned char raw_shared[];
  BackwardShared<T, Sh>& m = *reinterpret_cast<BackwardShared<T, Sh>*>(raw_shared);

  const ScanWhere at = scan_where(a);
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  const int sg = lane % GS, cell = warp * LC + lane / GS;
  const int c0 = at.ct * CT, left = a.per_group - c0;
  const int64_t cbase = int64_t(at.g) * a.per_group + c0;
  const int64_t len = scan_length(a, at.b);
  const int64_t first = int64_t(at.seg) * a.seg_tiles * kScanTile;
  const int64_t stop = min(first + int64_t(a.seg_tiles) * kScanTile, a.length);
  const int64_t live = max(min(stop, len), first);

  const int c_lane = CH * cell;
  Pairs<S> carry[CH], a2[CH], dA[CH];  // carry: a_{t+1} g_{t+1}
#pragma unroll
  for (int c = 0; c < CH; ++c)
#pragma unroll
    for (int s = 0; s < S; ++s) {
      const int n = sg * S + s;
      const bool on = n < a.states && c_lane + c < left;
      const int64_t i = (cbase + c_lane + c) * a.states + n;
      (s % 2 ? a2[c].v[s / 2].y : a2[c].v[s / 2].x) = on ? a.A[i] * kLog2e : 0.f;
      (s % 2 ? carry[c].v[s / 2].y : carry[c].v[s / 2].x) =
          on && a.dfinal ? a.dfinal[at.b * a.channels * a.states + i] : 0.f;
      (s % 2 ? dA[c].v[s / 2].y : dA[c].v[s / 2].x) = 0.f;
    }
  const int col = Share::col();
  float skip[V], bias[V], dD[V], dbias[V];
#pragma unroll
  for (int i = 0; i < V; ++i) {
    skip[i] = a.D && col + i < left ? a.D[cbase + col + i] : 0.f;
    bias[i] = a.dbias && col + i < left ? a.dbias[cbase + col + i] : 0.f;
    dD[i] = dbias[i] = 0.f;
  }
  const int64_t dense = at.b * a.length * a.channels + cbase + col;  // of the contiguous gradients
  T* du = static_cast<T*>(a.du) + dense;
  T* ddl = static_cast<T*>(a.ddelta) + dense;
  T* dz = static_cast<T*>(a.dz) + dense;
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

  auto fetch = [&](int64_t t0, int slot) {
    const T* u = static_cast<const T*>(a.u) + at.b * a.ub + cbase + col;
    const T* dl = static_cast<const T*>(a.delta) + at.b * a.db + cbase + col;
    const T* z = static_cast<const T*>(a.z) + at.b * a.zb + cbase + col;
    const T* dy = static_cast<const T*>(a.dy) + at.b * a.dyb + cbase + col;
    const T* B = static_cast<const T*>(a.B) + at.b * a.Bb + at.g * a.Bg;
    const T* C = static_cast<const T*>(a.C) + at.b * a.Cb + at.g * a.Cg;
#pragma unroll
    for (int i = 0; i < CNT; ++i) {
      const int64_t t = t0 + Share::row(i);
      const int n = t < live ? left - col : 0;
      stage_chunk<T, V>(&m.raw[slot][0][i][threadIdx.x], u + t * a.us, static_cast<const T*>(a.u), n, a.mode_act);
      stage_chunk<T, V>(&m.raw[slot][1][i][threadIdx.x], dl + t * a.ds, static_cast<const T*>(a.delta), n, a.mode_act);
      if (a.z)
        stage_chunk<T, V>(&m.raw[slot][2][i][threadIdx.x], z + t * a.zs, static_cast<const T*>(a.z), n, a.mode_act);
      stage_chunk<T, V>(&m.raw[slot][3][i][threadIdx.x], dy + t * a.dys, static_cast<const T*>(a.dy), n, a.mode_act);
    }
#pragma unroll
    for (int i = 0; i < States::CNT; ++i) {
      const int k = States::item(i), n = States::state(k);
      const int64_t t = t0 + States::row(k);
      const int on = k < States::ITEMS && t < live ? a.states - n : 0;
      stage_chunk<T, VB>(&m.raw_bc[slot][0][i][threadIdx.x], B + t * a.Bs + n, B, on, a.mode_bc);
      stage_chunk<T, VB>(&m.raw_bc[slot][1][i][threadIdx.x], C + t * a.Cs + n, C, on, a.mode_bc);
    }
  };
  const int64_t tiles = (live - first + kScanTile - 1) / kScanTile;
  if (tiles > 0) fetch(first + (tiles - 1) * kScanTile, 0);
  copy_commit();
  int slot = 0;
  for (int64_t tile = tiles - 1; tile >= 0; --tile, slot ^= 1) {
    const int64_t t0 = first + tile * kScanTile;
    Pairs<S> h0[CH], h[kScanTile][CH];
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      const float* k = a.saved + ((at.b * ((a.length + kScanTile - 1) / kScanTile) + t0 / kScanTile) * a.channels +
                                  cbase + c_lane + c) * NP + sg * S;
      if (c_lane + c < left) h0[c] = *reinterpret_cast<const Pairs<S>*>(k);
      else h0[c] = Pairs<S>{};
    }
    if (tile > 0) fetch(t0 - kScanTile, slot ^ 1);  // the next one to work on
    copy_commit();
    copy_wait<1>();
#pragma unroll
    for (int i = 0; i < CNT; ++i) {
      const int r = Share::row(i);
      const int n = t0 + r < live ? left - col : 0;
      const Chunk<T, V> cu = m.raw[slot][0][i][threadIdx.x], cd = m.raw[slot][1][i][threadIdx.x],
                        cz = m.raw[slot][2][i][threadIdx.x], cy = m.raw[slot][3][i][threadIdx.x];
      float d[V], x[V], e[V];
#pragma unroll
      for (int j = 0; j < V; ++j) d[j] = to_f(cd.v[j]) + bias[j];
      if (a.softplus) by_two<V>(d, softplus, softplus2);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        d[j] = j < n ? d[j] : 0.f;
        x[j] = d[j] * to_f(cu.v[j]);
        e[j] = to_f(cz.v[j]);
      }
      put_steps<CH, V>(m.step[r], col, d, x);
      if (a.z) by_two<V>(e, [](float v) { return v * sigmoid(v); }, [](float2 v) { return mul2(v, sigmoid2(v)); });
#pragma unroll
      for (int j = 0; j < V; ++j) m.e[r][col + j] = a.z ? e[j] * to_f(cy.v[j]) : to_f(cy.v[j]);
    }
#pragma unroll
    for (int i = 0; i < States::CNT; ++i) {
      const int k = States::item(i);
      if (k < States::ITEMS) {
        const Chunk<T, VB> cb = m.raw_bc[slot][0][i][threadIdx.x], cc = m.raw_bc[slot][1][i][threadIdx.x];
#pragma unroll
        for (int j = 0; j < VB; ++j) {
          m.B[States::row(k)][States::state(k) + j] = to_f(cb.v[j]);
          m.C[States::row(k)][States::state(k) + j] = to_f(cc.v[j]);
        }
      }
    }
    __syncthreads();

    // The tile's states, and sum_n C h for the gate's gradient.
    constexpr int UY = GS > CH ? GS / CH : 1, OY = UY * CH / GS;
#pragma unroll
    for (int r0 = 0; r0 < kScanTile; r0 += UY) {
      float v[UY * CH];
#pragma unroll
      for (int j = 0; j < UY; ++j) {
        const int r = r0 + j;
        const Step<CH> st = m.step[r][cell];
        const Pairs<S> Bn = *reinterpret_cast<const Pairs<S>*>(&m.B[r][sg * S]);
        const Pairs<S> Cn = *reinterpret_cast<const Pairs<S>*>(&m.C[r][sg * S]);
#pragma unroll
        for (int c = 0; c < CH; ++c) {
          float2 acc = make_float2(0.f, 0.f);
#pragma unroll
          for (int s = 0; s < S / 2; ++s) {
            const float2 before = r == 0 ? h0[c].v[s] : h[r > 0 ? r - 1 : 0][c].v[s];
            const float2 x = decay(both(st.d[c]), a2[c].v[s]);
            h[r][c].v[s] = fma2(x, before, mul2(both(st.du[c]), Bn.v[s]));
            acc = fma2(h[r][c].v[s], Cn.v[s], acc);
          }
          v[j * CH + c] = acc.x + acc.y;
        }
      }
      if (a.z) {
        reduce_scatter<UY * CH, GS, 1>(v, lane);
#pragma unroll
        for (int i = 0; i < OY; ++i) {
          const int id = sg * OY + i;
          m.sum_y[r0 + id / CH][c_lane + id % CH] = v[i];
        }
      }
    }

    // Backwards.  UG steps share the sums over states (2 CH values a step), UB those over channels (2 S).
    constexpr int UG = GS > 2 * CH ? GS / (2 * CH) : 1, NG = 2 * CH * UG / GS;
    constexpr int UB = LC > 2 * S ? LC / (2 * S) : 1, NB = 2 * S * UB / LC;
    constexpr int UU = UG > UB ? UG : UB;
#pragma unroll
    for (int r0 = kScanTile - UU; r0 >= 0; r0 -= UU) {
      float vg[UU][2 * CH], vb[UU][2 * S];
#pragma unroll
      for (int j = UU - 1; j >= 0; --j) {
        const int r = r0 + j;
        const Step<CH> st = m.step[r][cell];
        const Pairs<S> Bn = *reinterpret_cast<const Pairs<S>*>(&m.B[r][sg * S]);
        const Pairs<S> Cn = *reinterpret_cast<const Pairs<S>*>(&m.C[r][sg * S]);
        Pairs<S> db, dc;
#pragma unroll
        for (int c = 0; c < CH; ++c) {
          const float2 e = both(m.e[r][c_lane + c]), d = both(st.d[c]), x = both(st.du[c]);
          float2 g2 = make_float2(0.f, 0.f), w2 = make_float2(0.f, 0.f);
#pragma unroll
          for (int s = 0; s < S / 2; ++s) {
            const float2 ex = decay(d, a2[c].v[s]);
            const float2 before = r == 0 ? h0[c].v[s] : h[r > 0 ? r - 1 : 0][c].v[s];
            const float2 g = fma2(Cn.v[s], e, carry[c].v[s]);
            carry[c].v[s] = mul2(ex, g);
            const float2 w = mul2(carry[c].v[s], before);
            w2 = fma2(w, a2[c].v[s], w2);
            dA[c].v[s] = fma2(w, d, dA[c].v[s]);
            g2 = fma2(g, Bn.v[s], g2);
            db.v[s] = c == 0 ? mul2(g, x) : fma2(g, x, db.v[s]);
            dc.v[s] = c == 0 ? mul2(h[r][c].v[s], e) : fma2(h[r][c].v[s], e, dc.v[s]);
          }
          vg[j][2 * c] = g2.x + g2.y;
          vg[j][2 * c + 1] = w2.x + w2.y;
        }
#pragma unroll
        for (int s = 0; s < S / 2; ++s) {
          vb[j][2 * s] = db.v[s].x;
          vb[j][2 * s + 1] = db.v[s].y;
          vb[j][S + 2 * s] = dc.v[s].x;
          vb[j][S + 2 * s + 1] = dc.v[s].y;
        }
      }
#pragma unroll
      for (int q = 0; q < UU / UG; ++q) {
        float v[2 * CH * UG];
#pragma unroll
        for (int i = 0; i < 2 * CH * UG; ++i) v[i] = vg[q * UG + i / (2 * CH)][i % (2 * CH)];
        reduce_scatter<2 * CH * UG, GS, 1>(v, lane);
#pragma unroll
        for (int i = 0; i < NG; ++i) {
          const int id = sg * NG + i, r = r0 + q * UG + id / (2 * CH), k = id % (2 * CH);
          (k % 2 ? m.sum_w : m.sum_g)[r][c_lane + k / 2] = v[i];
        }
      }
#pragma unroll
      for (int q = 0; q < UU / UB; ++q) {
        float v[2 * S * UB];
#pragma unroll
        for (int i = 0; i < 2 * S * UB; ++i) v[i] = vb[q * UB + i / (2 * S)][i % (2 * S)];
        reduce_scatter<2 * S * UB, LC, GS>(v, lane);
#pragma unroll
        for (int i = 0; i < NB; ++i) {
          const int id = lane / GS * NB + i, r = r0 + q * UB + id / (2 * S), k = id % (2 * S);
          m.bc[warp][r][k / S * NP + sg * S + k % S] = v[i];
        }
      }
    }
    __syncthreads();

#pragma unroll
    for (int i = 0; i < CNT; ++i) {
      const int r = Share::row(i);
      const int64_t t = t0 + r;
      if (t >= stop) continue;
      const Chunk<T, V> cu = m.raw[slot][0][i][threadIdx.x], cd = m.raw[slot][1][i][threadIdx.x],
                        cz = m.raw[slot][2][i][threadIdx.x], cy = m.raw[slot][3][i][threadIdx.x];
      Chunk<T, V> ou, od, oz;
      float slope[V];
#pragma unroll
      for (int j = 0; j < V; ++j) slope[j] = to_f(cd.v[j]) + bias[j];
      if (a.softplus) by_two<V>(slope, sigmoid, sigmoid2);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float uf = to_f(cu.v[j]);
        const float e = m.e[r][col + j], d = m.step[r][(col + j) / CH].d[(col + j) % CH], gB = m.sum_g[r][col + j];
        float dd = fmaf(m.sum_w[r][col + j], kLn2, gB * uf);
        if (a.softplus) dd *= slope[j];
        if (t >= live) dd = 0.f;
        ou.v[j] = from_f<T>(fmaf(d, gB, skip[j] * e));
        od.v[j] = from_f<T>(dd);
        dD[j] = fmaf(e, uf, dD[j]);
        dbias[j] += dd;
      }
      store_chunk<T, V>(du + t * a.channels, ou, left - col, a.vec);
      store_chunk<T, V>(ddl + t * a.channels, od, left - col, a.vec);
      if (a.z) {
        float s[V];
#pragma unroll
        for (int j = 0; j < V; ++j) s[j] = to_f(cz.v[j]);
        by_two<V>(s, sigmoid, sigmoid2);
#pragma unroll
        for (int j = 0; j < V; ++j)
          oz.v[j] = from_f<T>(to_f(cy.v[j]) * fmaf(skip[j], to_f(cu.v[j]), m.sum_y[r][col + j]) *
                              (s[j] * fmaf(to_f(cz.v[j]), 1.f - s[j], 1.f)));
        store_chunk<T, V>(dz + t * a.channels, oz, left - col, a.vec);
      }
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
    for (int c = 0; c < CH; ++c)
#pragma unroll
      for (int s = 0; s < S; ++s) {
        const int n = sg * S + s;
        if (n < a.states && c_lane + c < left)
          a.dinit[(at.b * a.channels + cbase + c_lane + c) * a.states + n] =
              s % 2 ? carry[c].v[s / 2].y : carry[c].v[s / 2].x;
      }
  }
  const int64_t prow = (at.b * a.segments + at.seg) * a.channels + cbase;
#pragma unroll
  for (int c = 0; c < CH; ++c)
    if (c_lane + c < left) *reinterpret_cast<Pairs<S>*>(a.part_a + (prow + c_lane + c) * NP + sg * S) = dA[c];
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
    case 4: return f(ScanShape<2, 2, 2, 2>{});
    case 8: return f(ScanShape<4, 2, 2, 2>{});
    case 16: return f(ScanShape<4, 2, 4, 4>{});
    case 32: return f(ScanShape<4, 2, 8, 4>{});
    default: return f(ScanShape<4, 2, 16, 4>{});
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
  constexpr int smem = int(sizeof(BackwardShared<T, Sh>));
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
  const uint64_t es = uint64_t(layer_elem_size(d->dtype));
  auto at = [](const void* p) { return uint64_t(reinterpret_cast<uintptr_t>(p)); };
  a.mode_act = copy_mode(at(u) | at(delta) | at(z) | at(dy) |
                         es * (a.per_group | a.ub | a.us | a.db | a.ds | (z ? a.zb | a.zs : 0) | a.dyb | a.dys));
  a.mode_bc = copy_mode((at(B) | at(C) | es * (a.states | a.Bb | a.Bs | a.Bg | a.Cb | a.Cs | a.Cg)) % 4 ? 1 : 4);
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
