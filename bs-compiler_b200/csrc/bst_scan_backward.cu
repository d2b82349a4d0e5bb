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
// Two exponentials for each (position, channel, state) and the sums over states and over channels that
// each step asks for bound it: they go through reduce_scatter over the lanes, dB and dC then through
// shared memory over the block's warps and through a partial array over the channel tiles.
//
// Measured on B200, 4 x 2048 x 4096 with 16 states in bf16: 983 us and 17 us for the sums over the channel tiles
// (29 instructions per (position, channel, state) before the series near 1 was added, schedulers 50 % busy at two
// warps each: the 16 states of a tile take 128 registers).
#include <algorithm>

#include "bst_scan.cuh"

namespace bst {

template <typename T, class Sh>
struct BackwardShared {
  alignas(128) T act[2][4][kScanTile][Sh::CT];                    // u, delta, dy, z as they come: this tile, the next
  alignas(128) T bc[2][2][kScanTile][Sh::NP];                     // B, C
  alignas(16) float d[kScanTile][Sh::CT], e[kScanTile][Sh::CT];   // step sizes, gradients of the sums over states
  alignas(16) float sum_y[kScanTile][Sh::CT];                     // sum_n C h
  float sum_g[kScanTile][Sh::CT], sum_w[kScanTile][Sh::CT];       // sum_n g B, sum_n A log2(e) w
  float part[Sh::W][kScanTile][2 * Sh::NP];                       // per warp: dB, dC summed over its channels
  uint64_t bar[2];
};

template <typename T, class Sh, bool TILES>
__global__ void __launch_bounds__(Sh::NT) scan_backward_kernel(const ScanArgs a,
                                                               const __grid_constant__ ScanMaps maps) {
  constexpr int S = Sh::S, CH = Sh::CH, GS = Sh::GS, CT = Sh::CT, NP = Sh::NP, NT = Sh::NT, W = Sh::W;
  constexpr int LC = 32 / GS;  // lanes of a warp that share a state group
  constexpr int PAIRS = CT / 2, ROWS = NT / PAIRS, TURNS = kScanTile / ROWS;
  extern __shared__ __align__(128) unsigned char raw_shared[];
  BackwardShared<T, Sh>& m = *reinterpret_cast<BackwardShared<T, Sh>*>(raw_shared);

  const ScanWhere at = scan_where(a);
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  const int sg = lane % GS, cell = warp * LC + lane / GS;
  const int c0 = at.ct * CT, left = a.per_group - c0, cols = left < CT ? left : CT;
  const int64_t cbase = int64_t(at.g) * a.per_group + c0;
  const int64_t len = scan_length(a, at.b);
  const int tiles = int((len + kScanTile - 1) / kScanTile);

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
  // Outside of the recurrences a thread has a pair of neighbouring channels and every ROWS-th position.
  const int col = threadIdx.x % PAIRS * 2, row0 = threadIdx.x / PAIRS;
  const bool in0 = col < left, in1 = col + 1 < left;
  float2 skip = both(0.f), bias = both(0.f), dD = both(0.f), dbias = both(0.f);
  if (a.D) skip = make_float2(in0 ? a.D[cbase + col] : 0.f, in1 ? a.D[cbase + col + 1] : 0.f);
  if (a.dbias) bias = make_float2(in0 ? a.dbias[cbase + col] : 0.f, in1 ? a.dbias[cbase + col + 1] : 0.f);
  const int64_t dense = at.b * a.length * a.channels + cbase + col;  // of the contiguous gradients
  T* du = static_cast<T*>(a.du) + dense;
  T* ddl = static_cast<T*>(a.ddelta) + dense;
  T* dz = static_cast<T*>(a.dz) + dense;
  float* part = a.part_bc + ((at.b * a.groups + at.g) * a.col_tiles + at.ct) * a.length * 2 * NP;

  // Positions behind the sequence's end.
  for (int64_t t = int64_t(tiles) * kScanTile + row0; t < a.length; t += ROWS) {
    const Chunk<T, 2> zero = to_pair<T>(both(0.f));
    store_chunk<T, 2>(du + t * a.channels, zero, left - col, a.vec);
    store_chunk<T, 2>(ddl + t * a.channels, zero, left - col, a.vec);
    if (a.dz) store_chunk<T, 2>(dz + t * a.channels, zero, left - col, a.vec);
  }

  bool failed = false;
  if (TILES) {
    if (threadIdx.x == 0) {
      mbar_init(&m.bar[0], 1);
      mbar_init(&m.bar[1], 1);
      mbar_fence_init();
    }
    __syncthreads();
  }
  auto fetch = [&](int k, int slot) {
    if (k >= 0) {
      auto& act = m.act[slot];
      auto& bc = m.bc[slot];
      const int64_t t0 = int64_t(k) * kScanTile;
      if constexpr (TILES) {
        if (threadIdx.x == 0) {
          uint64_t* bar = &m.bar[slot];
          const int t = int(t0), c = int(cbase), b = int(at.b);
          mbar_expect_tx(bar, unsigned((a.z ? 4 : 3) * sizeof(act[0]) + sizeof(bc)));
          tma_load_3d(&act[0][0][0], &maps.u, bar, c, t, b);
          tma_load_3d(&act[1][0][0], &maps.delta, bar, c, t, b);
          tma_load_3d(&act[2][0][0], &maps.dy, bar, c, t, b);
          if (a.z) tma_load_3d(&act[3][0][0], &maps.z, bar, c, t, b);
          tma_load_4d(&bc[0][0][0], &maps.B, bar, 0, at.g, t, b);
          tma_load_4d(&bc[1][0][0], &maps.C, bar, 0, at.g, t, b);
        }
      } else {
        const int rows = int(min(len - t0, int64_t(kScanTile))), me = threadIdx.x;
        const bool words = a.mode == kCopyWords;
        auto stage = [&](auto width, T* to, const void* p, int64_t off, int64_t st, int n) {
          stage_tile<T, decltype(width)::value, NT>(to, static_cast<const T*>(p) + off + t0 * st, st, rows, n, words, me);
        };
        std::integral_constant<int, CT> wide;
        std::integral_constant<int, NP> slim;
        stage(wide, &act[0][0][0], a.u, at.b * a.ub + cbase, a.us, cols);
        stage(wide, &act[1][0][0], a.delta, at.b * a.db + cbase, a.ds, cols);
        stage(wide, &act[2][0][0], a.dy, at.b * a.dyb + cbase, a.dys, cols);
        if (a.z) stage(wide, &act[3][0][0], a.z, at.b * a.zb + cbase, a.zs, cols);
        stage(slim, &bc[0][0][0], a.B, at.b * a.Bb + at.g * a.Bg, a.Bs, a.states);
        stage(slim, &bc[1][0][0], a.C, at.b * a.Cb + at.g * a.Cg, a.Cs, a.states);
      }
    }
    if constexpr (!TILES) copy_commit();
  };
  fetch(tiles - 1, 0);
  int slot = 0, turn = 0;
  for (int k = tiles - 1; k >= 0; --k) {
    const int64_t t0 = int64_t(k) * kScanTile;
    const int rows = int(min(len - t0, int64_t(kScanTile)));
    Pairs<S> h0[CH], h[kScanTile][CH];
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      const float* p = a.saved + ((at.b * ((a.length + kScanTile - 1) / kScanTile) + t0 / kScanTile) * a.channels +
                                  cbase + c_lane + c) * NP + sg * S;
      if (c_lane + c < left) h0[c] = *reinterpret_cast<const Pairs<S>*>(p);
      else h0[c] = Pairs<S>{};
    }
    fetch(k - 1, slot ^ 1);  // the next tile to work on
    if constexpr (TILES) {
      if (!failed && !mbar_wait_bounded(&m.bar[slot], unsigned(turn) & 1u)) {
        failed = true;
        atomicOr(a.error, kErrTmaTimeout);
      }
    } else {
      copy_wait<1>();
      __syncthreads();  // everybody's copies
    }
    auto& act = m.act[slot];
    {
      float2 d[TURNS], e[TURNS];
#pragma unroll
      for (int i = 0; i < TURNS; ++i) {
        d[i] = add2(load_pair(&act[1][row0 + i * ROWS][col]), bias);
        e[i] = load_pair(&act[2][row0 + i * ROWS][col]);
      }
      if (a.softplus) {
#pragma unroll
        for (int i = 0; i < TURNS; ++i) d[i] = softplus2(d[i]);
      }
      if (a.z) {
#pragma unroll
        for (int i = 0; i < TURNS; ++i) {
          const float2 z = load_pair(&act[3][row0 + i * ROWS][col]);
          e[i] = mul2(e[i], mul2(z, sigmoid2(z)));
        }
      }
      if (rows < kScanTile) {  // what lies behind the sequence's end may be anything: it becomes zeros
#pragma unroll
        for (int i = 0; i < TURNS; ++i)
          if (row0 + i * ROWS >= rows) {
            d[i] = e[i] = both(0.f);
            *reinterpret_cast<Chunk<T, 2>*>(&act[0][row0 + i * ROWS][col]) = to_pair<T>(both(0.f));
          }
        for (int j = rows * NP + int(threadIdx.x); j < kScanTile * NP; j += NT)
          (&m.bc[slot][0][0][0])[j] = (&m.bc[slot][1][0][0])[j] = from_f<T>(0.f);
        if constexpr (TILES) fence_proxy_async_smem();  // before the copy engine writes to this slot again
      }
#pragma unroll
      for (int i = 0; i < TURNS; ++i) {
        *reinterpret_cast<float2*>(&m.d[row0 + i * ROWS][col]) = d[i];
        *reinterpret_cast<float2*>(&m.e[row0 + i * ROWS][col]) = e[i];
      }
    }
    __syncthreads();

    // What a step of the recurrences reads.
    struct Operands {
      Chunk<float, CH> d, e;
      Chunk<T, CH> u;
      Chunk<T, S> B, C;
    };
    auto load = [&](int r) {
      Operands o;
      o.d = *reinterpret_cast<const Chunk<float, CH>*>(&m.d[r][c_lane]);
      o.e = *reinterpret_cast<const Chunk<float, CH>*>(&m.e[r][c_lane]);
      o.u = *reinterpret_cast<const Chunk<T, CH>*>(&act[0][r][c_lane]);
      o.B = *reinterpret_cast<const Chunk<T, S>*>(&m.bc[slot][0][r][sg * S]);
      o.C = *reinterpret_cast<const Chunk<T, S>*>(&m.bc[slot][1][r][sg * S]);
      return o;
    };
    // The tile's states, and sum_n C h for the gate's gradient (left in registers until the loop is over: a store
    // in between would hold back the loads of the later steps).
    constexpr int UY = GS > CH ? GS / CH : 1, OY = UY * CH / GS;
    float sums[kScanTile / UY][OY];
#pragma unroll
    for (int r0 = 0; r0 < kScanTile; r0 += UY) {
      float v[UY * CH];
#pragma unroll
      for (int j = 0; j < UY; ++j) {
        const int r = r0 + j;
        const Operands o = load(r);
        const Pairs<S> Bn = load_states<S>(o.B.v), Cn = load_states<S>(o.C.v);
#pragma unroll
        for (int c = 0; c < CH; ++c) {
          const float x = o.d.v[c] * to_f(o.u.v[c]);
          float2 acc = make_float2(0.f, 0.f);
#pragma unroll
          for (int s = 0; s < S / 2; ++s) {
            const float2 before = r == 0 ? h0[c].v[s] : h[r > 0 ? r - 1 : 0][c].v[s];
            h[r][c].v[s] = fma2(decay(both(o.d.v[c]), a2[c].v[s]), before, mul2(both(x), Bn.v[s]));
            acc = s == 0 ? mul2(h[r][c].v[s], Cn.v[s]) : fma2(h[r][c].v[s], Cn.v[s], acc);
          }
          v[j * CH + c] = acc.x + acc.y;
        }
      }
      if (a.z) reduce_scatter<UY * CH, GS, 1>(v, lane);
#pragma unroll
      for (int i = 0; i < OY; ++i) sums[r0 / UY][i] = v[i];
    }
    if (a.z) {
#pragma unroll
      for (int r0 = 0; r0 < kScanTile; r0 += UY)
#pragma unroll
        for (int i = 0; i < OY; ++i) {
          const int id = sg * OY + i;
          m.sum_y[r0 + id / CH][c_lane + id % CH] = sums[r0 / UY][i];
        }
    }

    // Backwards.  UG steps share the sums over states (2 CH values a step), UB those over channels (2 S).  The
    // operands are loaded AHEAD steps early, past the stores of the steps in between.
    constexpr int UG = GS > 2 * CH ? GS / (2 * CH) : 1, NG = 2 * CH * UG / GS;
    constexpr int UB = LC > 2 * S ? LC / (2 * S) : 1, NB = 2 * S * UB / LC;
    constexpr int UU = UG > UB ? UG : UB;
    constexpr int AHEAD = UU > 2 ? UU : 2;
    Operands next[AHEAD];
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) next[j] = load(kScanTile - 1 - j);
#pragma unroll
    for (int r0 = kScanTile - UU; r0 >= 0; r0 -= UU) {
      float vg[UU][2 * CH], vb[UU][2 * S];
#pragma unroll
      for (int j = UU - 1; j >= 0; --j) {
        const int r = r0 + j;
        const Operands o = next[(kScanTile - 1 - r) % AHEAD];
        if (r >= AHEAD) next[(kScanTile - 1 - r) % AHEAD] = load(r - AHEAD);
        const Pairs<S> Bn = load_states<S>(o.B.v), Cn = load_states<S>(o.C.v);
        Pairs<S> db, dc;
#pragma unroll
        for (int c = 0; c < CH; ++c) {
          const float2 e = both(o.e.v[c]), d = both(o.d.v[c]), x = both(o.d.v[c] * to_f(o.u.v[c]));
          float2 g2 = make_float2(0.f, 0.f), w2 = make_float2(0.f, 0.f);
#pragma unroll
          for (int s = 0; s < S / 2; ++s) {
            const float2 before = r == 0 ? h0[c].v[s] : h[r > 0 ? r - 1 : 0][c].v[s];
            const float2 g = fma2(Cn.v[s], e, carry[c].v[s]);
            carry[c].v[s] = mul2(decay(d, a2[c].v[s]), g);
            const float2 w = mul2(carry[c].v[s], before);
            w2 = s == 0 ? mul2(w, a2[c].v[s]) : fma2(w, a2[c].v[s], w2);
            dA[c].v[s] = fma2(w, d, dA[c].v[s]);
            g2 = s == 0 ? mul2(g, Bn.v[s]) : fma2(g, Bn.v[s], g2);
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
          const int id = sg * NG + i, r = r0 + q * UG + id / (2 * CH), j = id % (2 * CH);
          (j % 2 ? m.sum_w : m.sum_g)[r][c_lane + j / 2] = v[i];
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
          const int id = lane / GS * NB + i, r = r0 + q * UB + id / (2 * S), j = id % (2 * S);
          m.part[warp][r][j / S * NP + sg * S + j % S] = v[i];
        }
      }
    }
    __syncthreads();

    {
      float2 x[TURNS], v[TURNS], slope[TURNS];
      // Values of this thread's positions, to be stored behind `to`: branches stand outside of the loops.
      const bool inside = a.vec && in1 && rows == kScanTile;
      auto put = [&](T* to) {
        T* p = to + (t0 + row0) * a.channels;
        const int64_t step = int64_t(ROWS) * a.channels;
        if (inside) {
#pragma unroll
          for (int i = 0; i < TURNS; ++i) *reinterpret_cast<Chunk<T, 2>*>(p + i * step) = to_pair<T>(v[i]);
        } else {
#pragma unroll
          for (int i = 0; i < TURNS; ++i)
            if (t0 + row0 + i * ROWS < a.length)
              store_chunk<T, 2>(p + i * step, to_pair<T>(v[i]), left - col, false);
        }
      };
#pragma unroll
      for (int i = 0; i < TURNS; ++i) {
        const int r = row0 + i * ROWS;
        const float2 e = *reinterpret_cast<const float2*>(&m.e[r][col]);
        x[i] = load_pair(&act[0][r][col]);
        dD = fma2(e, x[i], dD);
        v[i] = fma2(*reinterpret_cast<const float2*>(&m.d[r][col]), *reinterpret_cast<const float2*>(&m.sum_g[r][col]),
                    mul2(skip, e));
        slope[i] = both(1.f);
      }
      put(du);
      if (a.softplus) {
#pragma unroll
        for (int i = 0; i < TURNS; ++i) slope[i] = sigmoid2(add2(load_pair(&act[1][row0 + i * ROWS][col]), bias));
      }
#pragma unroll
      for (int i = 0; i < TURNS; ++i) {
        const int r = row0 + i * ROWS;
        const float2 w = *reinterpret_cast<const float2*>(&m.sum_w[r][col]);
        const float2 dd = mul2(slope[i], fma2(w, both(kLn2), mul2(*reinterpret_cast<const float2*>(&m.sum_g[r][col]),
                                                                  x[i])));
        v[i] = r < rows ? dd : both(0.f);
        dbias = add2(dbias, v[i]);
      }
      put(ddl);
      if (a.z) {
#pragma unroll
        for (int i = 0; i < TURNS; ++i) {
          const int r = row0 + i * ROWS;
          const float2 z = load_pair(&act[3][r][col]), s = sigmoid2(z);
          const float2 y = fma2(skip, x[i], *reinterpret_cast<const float2*>(&m.sum_y[r][col]));
          const float2 q = mul2(s, fma2(z, make_float2(1.f - s.x, 1.f - s.y), both(1.f)));
          v[i] = r < rows ? mul2(mul2(load_pair(&act[2][r][col]), y), q) : both(0.f);
        }
        put(dz);
      }
    }
    for (int j = threadIdx.x; j < kScanTile * 2 * NP; j += NT) {
      const int r = j / (2 * NP), n = j % (2 * NP);
      float v = 0.f;
#pragma unroll
      for (int i = 0; i < W; ++i) v += m.part[i][r][n];
      if (r < rows) part[(t0 + r) * 2 * NP + n] = v;
    }
    __syncthreads();
    if (slot) ++turn;
    slot ^= 1;
  }
  if (TILES && failed)  // copies that are late may not outlive the block
    for (int i = 0; i < 2; ++i) mbar_wait_bounded(&m.bar[i], unsigned(turn) & 1u);

  if (a.dinit) {
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
  const int64_t prow = at.b * a.channels + cbase;
#pragma unroll
  for (int c = 0; c < CH; ++c)
    if (c_lane + c < left) *reinterpret_cast<Pairs<S>*>(a.part_a + (prow + c_lane + c) * NP + sg * S) = dA[c];
  float4* buf = reinterpret_cast<float4*>(&m.d[0][0]);  // d, e and the sums hold 80 CT floats, this takes 4 NT
  static_assert(4 * NT <= 80 * CT, "room for the column sums");
  __syncthreads();
  buf[threadIdx.x] = make_float4(dD.x, dD.y, dbias.x, dbias.y);
  __syncthreads();
  if (threadIdx.x < PAIRS) {
    float4 s = buf[threadIdx.x];
    for (int r = 1; r < ROWS; ++r) {
      const float4 v = buf[threadIdx.x + r * PAIRS];
      s.x += v.x, s.y += v.y, s.z += v.z, s.w += v.w;
    }
    float* p = a.part_d + (prow + col) * 2;
    if (in0) p[0] = s.x, p[1] = s.z;
    if (in1) p[2] = s.y, p[3] = s.w;
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
    const int64_t step = a.length * 2 * np;
    int k = 0;
    for (; k + 16 <= a.col_tiles; k += 16) {  // loads in flight together, added in order
      float x[16];
#pragma unroll
      for (int j = 0; j < 16; ++j) x[j] = p[(k + j) * step];
#pragma unroll
      for (int j = 0; j < 16; ++j) v += x[j];
    }
    for (; k < a.col_tiles; ++k) v += p[k * step];
  }
  T* out = static_cast<T*>(n2 < np ? a.dB : a.dC);
  out[((b * a.length + t) * a.groups + g) * a.states + n] = from_f<T>(v);
}

// dA, dD, ddelta_bias: sums over the sequences.
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
// The block shape of a request, as f(ScanShape).  Two channels per lane need fewer instructions, one channel half of
// the registers for a tile's states and gives twice the warps, which pays until its blocks (three per SM) no longer
// fit at once: 384 channel-state pairs per scheduler.  16 states, two | one: 5 x 777 x 514 in fp32 311 | 210 us,
// 2 x 2048 x 4096 in bf16 930 | 640, 4 x 2048 x 4096, before the series near 1, 886 | 1125.
template <class F>
static auto with_backward_shape(const bst_scan_desc* d, F&& f) {
  const int64_t pairs = d->batch * d->channels * scan_pad(d->states) / (int64_t(sm_count()) * 4);
  switch (scan_pad(d->states)) {
    case 4: return f(ScanShape<2, 2, 2, 2>{});
    case 8: return f(ScanShape<2, 2, 4, 4>{});
    case 16: return pairs >= 384 ? f(ScanShape<4, 2, 4, 4>{}) : f(ScanShape<4, 1, 4, 4>{});
    case 32: return pairs >= 384 ? f(ScanShape<4, 2, 8, 4>{}) : f(ScanShape<4, 1, 8, 4>{});
    default: return f(ScanShape<4, 2, 16, 4>{});
  }
}

struct BackwardLayout {
  int64_t bc, pa, pd, total;  // byte offsets of part_bc (0), part_a, part_d
};
static BackwardLayout backward_layout(const bst_scan_desc* d) {
  const int64_t np = scan_pad(d->states);
  const int64_t ct = with_backward_shape(d, [](auto sh) { return int64_t(decltype(sh)::CT); });
  const int64_t per_group = d->channels / d->groups, tiles = (per_group + ct - 1) / ct;
  BackwardLayout l{};
  l.pa = d->batch * d->groups * tiles * d->length * 2 * np * 4;
  l.pd = l.pa + d->batch * d->channels * np * 4;
  l.total = l.pd + d->batch * d->channels * 2 * 4;
  return l;
}

int64_t scan_backward_workspace(const bst_scan_desc* d) { return backward_layout(d).total; }

template <typename T, class Sh>
static int scan_backward_launch(const bst_scan_desc* d, ScanArgs a, cudaStream_t st) {
  a.col_tiles = (a.per_group + Sh::CT - 1) / Sh::CT;
  const int64_t blocks = int64_t(a.batch) * a.groups * a.col_tiles;
  const int64_t outs = int64_t(a.batch) * a.length * a.groups * 2 * Sh::NP;
  if (blocks > INT_MAX || outs / 256 + 1 > INT_MAX)
    return fail(BST_ERR_UNSUPPORTED, "the scan's gradients need more than 2^31 blocks");
  constexpr int smem = int(sizeof(BackwardShared<T, Sh>));
  ScanMaps maps;
  if (a.mode == kCopyTiles && !scan_maps(d, Sh::CT, Sh::NP, a.u, a.delta, a.z, a.dy, a.B, a.C, &maps))
    a.mode = kCopyWords;
  auto* kernel = a.mode == kCopyTiles ? scan_backward_kernel<T, Sh, true> : scan_backward_kernel<T, Sh, false>;
  BST_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
  kernel<<<unsigned(blocks), Sh::NT, smem, st>>>(a, maps);
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
  if (!aligned16(saved)) return fail(BST_ERR_INVALID, "the saved states must be aligned to 16 bytes");
  if (!workspace || workspace_bytes < need || !aligned16(workspace))
    return fail(BST_ERR_INVALID, "the workspace must hold " + std::to_string(need) + " bytes, aligned to 16");
  ScanArgs a = scan_args(d);
  a.u = u, a.delta = delta, a.A = A, a.B = B, a.C = C, a.D = D, a.z = z, a.dbias = delta_bias, a.lengths = lengths;
  a.dy = dy, a.dfinal = dfinal, a.saved = static_cast<float*>(const_cast<void*>(saved));
  a.du = du, a.ddelta = ddelta, a.dB = dB, a.dC = dC, a.dz = z ? dz : nullptr, a.dinit = dinitial;
  const BackwardLayout l = backward_layout(d);
  char* ws = static_cast<char*>(workspace);
  a.part_bc = reinterpret_cast<float*>(ws);
  a.part_a = reinterpret_cast<float*>(ws + l.pa);
  a.part_d = reinterpret_cast<float*>(ws + l.pd);
  const int64_t per = 16 / layer_elem_size(d->dtype);
  a.vec = aligned16(u) && aligned16(delta) && aligned16(z) && aligned16(dy) && aligned16(du) && aligned16(ddelta) &&
          aligned16(dz) &&
          (a.per_group | a.ub | a.us | a.db | a.ds | (z ? a.zb | a.zs : 0) | a.dyb | a.dys) % per == 0;
  a.mode = scan_copy_mode(d, u, delta, z, dy, B, C);
  a.error = device_error_word();
  if (!a.error) return fail(BST_ERR_CUDA, "device error word unavailable");
  int rc = with_type(d->dtype, [&](auto t) {
    using T = decltype(t);
    return with_backward_shape(d, [&](auto sh) { return scan_backward_launch<T, decltype(sh)>(d, a, st); });
  });
  if (rc) return rc;
  const int np = scan_pad(d->states);
  const int64_t n = d->channels * (np + 2);
  scan_params_kernel<<<unsigned((n + 255) / 256), 256, 0, st>>>(a, np, a.batch, dA, dD, ddelta_bias);
  return launched("scan_params_kernel launch");
}
