// bst_scan.cu — selective scan: forward pass (bst_scan_forward) and workspace sizes.
//
// One exponential, a short series and four fused operations for each (position, channel, state): instruction issue
// and latency bound it, not HBM.  Measured on B200 with 16 states in bf16: 1 x 4096 x 4096 262 us and 4 x 2048 x 4096
// 325 us; the exponentials alone would take 60 and 119 us, the bytes 21 and 41.  Without the series near 1 it would
// be 188 and 250 us, and fp32 gradients of A would be twice as far off.
#include <algorithm>
#include <initializer_list>

#include "bst_scan.cuh"

namespace bst {

PFN_cuTensorMapEncodeTiled_v12000 tensor_map_encoder();  // bst_core.cu

// What the helpers copy into: tiles of u, delta, z and of B, C as they lie in memory.
template <typename T, class Sh>
struct ForwardRaw {
  static constexpr int SLOTS = 5;  // tile k is worked on, k + 1 and k + 2 converted, the others on their way
  alignas(128) T act[SLOTS][3][kScanTile][Sh::CT];
  alignas(128) T bc[SLOTS][2][kScanTile][Sh::NP];
  uint64_t bar[SLOTS];
};


// One block: CT channels of one sequence, its tiles in order.  The first half of its threads runs the
// recurrences.  The second half, its helpers, does all that is shared by the states: it copies the inputs in, two
// tiles ahead, turns them into step sizes, and after the recurrences of a tile adds D u, gates and stores y.
// Both sides work on different tiles at the same time (two buffers), so that the latencies of one are hidden by
// the other: few channels leave a scheduler with one or two recurrence warps.
template <typename T, class Sh, bool TILES>
__global__ void __launch_bounds__(2 * Sh::NT, 2)
    scan_forward_kernel(const ScanArgs a, const __grid_constant__ ScanMaps maps) {
  constexpr int S = Sh::S, CH = Sh::CH, GS = Sh::GS, CT = Sh::CT, NP = Sh::NP, NT = Sh::NT;
  using Raw = ForwardRaw<T, Sh>;
  constexpr int SLOTS = Raw::SLOTS;
  __shared__ __align__(16) float s_d[2][kScanTile][CT];  // step sizes
  __shared__ __align__(16) float s_y[2][kScanTile][CT];  // sum_n C h
  extern __shared__ __align__(128) unsigned char raw_shared[];
  Raw& raw = *reinterpret_cast<Raw*>(raw_shared);

  const ScanWhere at = scan_where(a);
  const int c0 = at.ct * CT, left = a.per_group - c0;  // channels of the group from this tile on
  const int64_t cbase = int64_t(at.g) * a.per_group + c0;
  const int64_t len = scan_length(a, at.b);
  const int tiles = int((len + kScanTile - 1) / kScanTile);

  if (threadIdx.x < NT) {
    const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
    const int sg = lane % GS, cell = warp * (32 / GS) + lane / GS, c_lane = CH * cell;
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
    for (int k = 0, slot = 0; k < tiles; ++k, slot = slot + 1 == SLOTS ? 0 : slot + 1) {
      const int buf = k & 1;
      if (a.saved) {
        float* p = a.saved + ((at.b * ((a.length + kScanTile - 1) / kScanTile) + k) * a.channels +
                              cbase + c_lane) * NP + sg * S;
#pragma unroll
        for (int c = 0; c < CH; ++c)
          if (c_lane + c < left) *reinterpret_cast<Pairs<S>*>(p + c * NP) = h[c];
      }
      bar_sync<2 * NT, kFull>(buf);
      constexpr int U = GS > CH ? GS / CH : 1;  // steps whose sums over the states are joined together
      constexpr int OUT = U * CH / GS;          // of which each lane ends with so many
      constexpr int Q = U > 2 ? U : 2;          // steps whose exponentials are under way together
      // The sums leave at the end: a store in between would hold back the loads of all later steps.
      float sums[kScanTile / U][OUT];
#pragma unroll
      for (int q0 = 0; q0 < kScanTile; q0 += Q) {
        Pairs<S> e[Q][CH], in[Q][CH];
#pragma unroll
        for (int j = 0; j < Q; ++j) {
          const Chunk<float, CH> d = *reinterpret_cast<const Chunk<float, CH>*>(&s_d[buf][q0 + j][c_lane]);
          const Chunk<T, CH> u = *reinterpret_cast<const Chunk<T, CH>*>(&raw.act[slot][0][q0 + j][c_lane]);
          const Pairs<S> Bn = load_states<S>(&raw.bc[slot][0][q0 + j][sg * S]);
#pragma unroll
          for (int c = 0; c < CH; ++c) {
            const float du = d.v[c] * to_f(u.v[c]);
#pragma unroll
            for (int s = 0; s < S / 2; ++s) {
              e[j][c].v[s] = decay(both(d.v[c]), a2[c].v[s]);
              in[j][c].v[s] = mul2(both(du), Bn.v[s]);
            }
          }
        }
#pragma unroll
        for (int r0 = q0; r0 < q0 + Q; r0 += U) {
          float v[U * CH];
#pragma unroll
          for (int j = 0; j < U; ++j) {
            const Pairs<S> Cn = load_states<S>(&raw.bc[slot][1][r0 + j][sg * S]);
#pragma unroll
            for (int c = 0; c < CH; ++c) {
              float2 acc = make_float2(0.f, 0.f);
#pragma unroll
              for (int s = 0; s < S / 2; ++s) {
                h[c].v[s] = fma2(e[r0 - q0 + j][c].v[s], h[c].v[s], in[r0 - q0 + j][c].v[s]);
                acc = s == 0 ? mul2(h[c].v[s], Cn.v[s]) : fma2(h[c].v[s], Cn.v[s], acc);
              }
              v[j * CH + c] = acc.x + acc.y;
            }
          }
          reduce_scatter<U * CH, GS, 1>(v, lane);
#pragma unroll
          for (int i = 0; i < OUT; ++i) sums[r0 / U][i] = v[i];
        }
      }
#pragma unroll
      for (int r0 = 0; r0 < kScanTile; r0 += U)
#pragma unroll
        for (int i = 0; i < OUT; ++i) {
          const int id = sg * OUT + i;
          s_y[buf][r0 + id / CH][c_lane + id % CH] = sums[r0 / U][i];
        }
      bar_arrive<2 * NT, kDone>(buf);
    }
    if (a.final_state) {
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
    return;
  }

  using Share = PairShare<Sh>;
  const int col = Share::col(), me = Share::me(), cols = left < CT ? left : CT;
  const bool in0 = col < left, in1 = col + 1 < left;
  const float2 skip = a.D ? make_float2(in0 ? a.D[cbase + col] : 0.f, in1 ? a.D[cbase + col + 1] : 0.f) : both(0.f);
  const float2 bias = a.dbias ? make_float2(in0 ? a.dbias[cbase + col] : 0.f, in1 ? a.dbias[cbase + col + 1] : 0.f)
                              : both(0.f);
  T* y = static_cast<T*>(a.y) + at.b * a.yb + cbase + col;

  int next = 0, next_slot = 0;  // the tile to fetch next, and where to
  bool failed = false;
  if constexpr (TILES) {
    if (me == 0) {
      for (int i = 0; i < SLOTS; ++i) mbar_init(&raw.bar[i], 1);
      mbar_fence_init();
    }
    bar_sync<NT, kHelp>(0);
  }
  auto fetch = [&] {
    if (next < tiles) {
      auto& act = raw.act[next_slot];
      auto& bc = raw.bc[next_slot];
      if constexpr (TILES) {
        if (me == 0) {
          uint64_t* bar = &raw.bar[next_slot];
          const int t = next * kScanTile, c = int(cbase), b = int(at.b);
          mbar_expect_tx(bar, unsigned((a.z ? 3 : 2) * sizeof(act[0]) + sizeof(bc)));
          tma_load_3d(&act[0][0][0], &maps.u, bar, c, t, b);
          tma_load_3d(&act[1][0][0], &maps.delta, bar, c, t, b);
          if (a.z) tma_load_3d(&act[2][0][0], &maps.z, bar, c, t, b);
          tma_load_4d(&bc[0][0][0], &maps.B, bar, 0, at.g, t, b);
          tma_load_4d(&bc[1][0][0], &maps.C, bar, 0, at.g, t, b);
        }
      } else {
        const int64_t t0 = int64_t(next) * kScanTile;
        const int rows = int(min(len - t0, int64_t(kScanTile)));
        const bool words = a.mode == kCopyWords;
        auto stage = [&](auto width, T* to, const void* p, int64_t off, int64_t st, int n) {
          stage_tile<T, decltype(width)::value, NT>(to, static_cast<const T*>(p) + off + t0 * st, st, rows, n, words, me);
        };
        std::integral_constant<int, CT> wide;
        std::integral_constant<int, NP> slim;
        stage(wide, &act[0][0][0], a.u, at.b * a.ub + cbase, a.us, cols);
        stage(wide, &act[1][0][0], a.delta, at.b * a.db + cbase, a.ds, cols);
        if (a.z) stage(wide, &act[2][0][0], a.z, at.b * a.zb + cbase, a.zs, cols);
        stage(slim, &bc[0][0][0], a.B, at.b * a.Bb + at.g * a.Bg, a.Bs, a.states);
        stage(slim, &bc[1][0][0], a.C, at.b * a.Cb + at.g * a.Cg, a.Cs, a.states);
      }
    }
    if constexpr (!TILES) copy_commit();  // one group per tile, empty behind the last
    ++next;
    next_slot = next_slot + 1 == SLOTS ? 0 : next_slot + 1;
  };
  // Waits for the tile in `slot`, its copy number `turn` into that slot (TILES), or for all but the last LEFT groups.
  auto arrived = [&](auto left_groups, int slot, int turn) {
    if constexpr (TILES) {
      if (!failed && !mbar_wait_bounded(&raw.bar[slot], unsigned(turn) & 1u)) {
        failed = true;
        atomicOr(a.error, kErrTmaTimeout);
      }
    } else {
      copy_wait<decltype(left_groups)::value>();
    }
  };
  constexpr int TURNS = Share::TURNS;
  struct Steps {
    float2 d[TURNS];
  };
  // The step sizes of tile k, computed into registers ahead of their turn.  In a tile that the sequence ends in, what
  // lies behind the end is cleared on the way, so that it meets the recurrences as zeros.
  auto convert = [&](int k, int slot) {
    Steps s;
    const int rows = int(min(len - int64_t(k) * kScanTile, int64_t(kScanTile)));
    // Every branch stands outside of the loops over the turns, whose latencies then overlap.
#pragma unroll
    for (int i = 0; i < TURNS; ++i) s.d[i] = add2(load_pair(&raw.act[slot][1][Share::row(i)][col]), bias);
    if (a.softplus) {
#pragma unroll
      for (int i = 0; i < TURNS; ++i) s.d[i] = softplus2(s.d[i]);
    }
    if (rows < kScanTile) {
#pragma unroll
      for (int i = 0; i < TURNS; ++i)
        if (Share::row(i) >= rows) {
          s.d[i] = both(0.f);
          *reinterpret_cast<Chunk<T, 2>*>(&raw.act[slot][0][Share::row(i)][col]) = to_pair<T>(both(0.f));
        }
      for (int j = rows * NP + me; j < kScanTile * NP; j += NT)
        (&raw.bc[slot][0][0][0])[j] = (&raw.bc[slot][1][0][0])[j] = from_f<T>(0.f);
    }
    return s;
  };
  // ... and handed over.
  auto publish = [&](const Steps& s, int buf) {
#pragma unroll
    for (int i = 0; i < TURNS; ++i) *reinterpret_cast<float2*>(&s_d[buf][Share::row(i)][col]) = s.d[i];
    bar_arrive<2 * NT, kFull>(buf);
  };
  std::integral_constant<int, SLOTS - 1> all_but_first;
  std::integral_constant<int, SLOTS - 2> all_but_two;
  std::integral_constant<int, SLOTS - 3> to_the_third;
#pragma unroll
  for (int k = 0; k < SLOTS; ++k) fetch();
  if (tiles > 0) {
    arrived(all_but_first, 0, 0);
    if constexpr (!TILES) bar_sync<NT, kHelp>(0);  // everybody's copies
    publish(convert(0, 0), 0);
  }
  if (tiles > 1) {
    arrived(all_but_two, 1, 0);
    if constexpr (!TILES) bar_sync<NT, kHelp>(0);
    publish(convert(1, 1), 1);
  }
  int slot = 0, ahead = 2, turn = 0;  // slots of tile k and k + 2, and the latter's turn
  for (int k = 0; k < tiles; ++k) {
    const int buf = k & 1;
    const int64_t t0 = int64_t(k) * kScanTile;
    // While the recurrences of tile k run: D u and the gate of tile k, the step sizes of tile k + 2.
    float2 v[TURNS], g[TURNS];
#pragma unroll
    for (int i = 0; i < TURNS; ++i) {
      v[i] = mul2(skip, load_pair(&raw.act[slot][0][Share::row(i)][col]));
      g[i] = both(1.f);
    }
    if (a.z) {
#pragma unroll
      for (int i = 0; i < TURNS; ++i) {
        const float2 z = load_pair(&raw.act[slot][2][Share::row(i)][col]);
        g[i] = mul2(z, sigmoid2(z));
      }
    }
    const bool more = k + 2 < tiles;
    Steps s;
    if (more || !TILES) arrived(to_the_third, ahead, turn);
    if constexpr (!TILES) bar_sync<NT, kHelp>(0);
    if (more) s = convert(k + 2, ahead);
    bar_sync<2 * NT, kDone>(buf);  // also: every helper has read the slot of tile k
#pragma unroll
    for (int i = 0; i < TURNS; ++i)
      v[i] = add2(v[i], *reinterpret_cast<const float2*>(&s_y[buf][Share::row(i)][col]));
    if (more) publish(s, buf);
    fetch();
#pragma unroll
    for (int i = 0; i < TURNS; ++i) v[i] = a.z ? mul2(v[i], g[i]) : v[i];
    T* row = y + (t0 + me / Share::PAIRS) * a.ys;
    if (a.vec && in1 && t0 + kScanTile <= len) {
#pragma unroll
      for (int i = 0; i < TURNS; ++i)
        *reinterpret_cast<Chunk<T, 2>*>(row + i * Share::ROWS * a.ys) = to_pair<T>(v[i]);
    } else {
#pragma unroll
      for (int i = 0; i < TURNS; ++i) {
        const int64_t t = t0 + Share::row(i);
        if (t < a.length)
          store_chunk<T, 2>(row + i * Share::ROWS * a.ys, to_pair<T>(t < len ? v[i] : both(0.f)), left - col, false);
      }
    }
    slot = slot + 1 == SLOTS ? 0 : slot + 1;
    if (++ahead == SLOTS) ahead = 0, ++turn;
  }
  if (TILES && failed)  // copies that are late may not outlive the block
    for (int i = 0; i < SLOTS; ++i) mbar_wait_bounded(&raw.bar[i], unsigned((next - 1 - i) / SLOTS) & 1u);
  // Positions behind the sequence's end.
  for (int64_t t = int64_t(tiles) * kScanTile + me / Share::PAIRS; t < a.length; t += Share::ROWS)
    store_chunk<T, 2>(y + t * a.ys, to_pair<T>(both(0.f)), left - col, a.vec);
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
  return a;
}

int64_t scan_saved_bytes(const bst_scan_desc* d) {
  return d->batch * ((d->length + kScanTile - 1) / kScanTile) * d->channels * scan_pad(d->states) * 4;
}

int64_t scan_backward_workspace(const bst_scan_desc* d);  // bst_scan_backward.cu

// The tensor copy engine needs 16-byte aligned rows of real (non-zero, forward) strides.
int scan_copy_mode(const bst_scan_desc* d, const void* u, const void* delta, const void* z, const void* dy,
                   const void* B, const void* C) {
  const int64_t es = layer_elem_size(d->dtype);
  uint64_t bits = uint64_t(es * (d->channels / d->groups)) | uint64_t(es * d->states);
  bool plain = true;  // strides that a tensor map can hold
  auto take = [&](const void* p, std::initializer_list<int64_t> strides) {
    if (!p) return;
    bits |= uint64_t(reinterpret_cast<uintptr_t>(p));
    for (int64_t s : strides) {
      bits |= uint64_t(s * es);
      plain = plain && s > 0 && s * es < (int64_t(1) << 40);
    }
  };
  take(u, {d->u_batch, d->u_step});
  take(delta, {d->delta_batch, d->delta_step});
  take(z, {d->z_batch, d->z_step});
  take(dy, {d->dy_batch, d->dy_step});
  take(B, {d->B_batch, d->B_step, d->B_group});
  take(C, {d->C_batch, d->C_step, d->C_group});
  if (bits % 16 == 0 && plain) return kCopyTiles;
  return bits % 4 == 0 ? kCopyWords : kCopyPlain;
}

bool scan_maps(const bst_scan_desc* d, int tile_channels, int pad, const void* u, const void* delta, const void* z,
               const void* dy, const void* B, const void* C, ScanMaps* m) {
  const auto encode = tensor_map_encoder();
  if (!encode) return false;
  const CUtensorMapDataType type = d->dtype == BST_F32    ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                   : d->dtype == BST_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                                          : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  const cuuint64_t es = cuuint64_t(layer_elem_size(d->dtype));
  const cuuint32_t ones[4] = {1, 1, 1, 1};
  auto one = [&](CUtensorMap* map, int rank, const void* p, const cuuint64_t* dims, const cuuint64_t* strides,
                 const cuuint32_t* box) {
    return encode(map, type, rank, const_cast<void*>(p), dims, strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE,
                  CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
  };
  auto act = [&](CUtensorMap* map, const void* p, int64_t batch, int64_t step) {
    const cuuint64_t dims[3] = {cuuint64_t(d->channels), cuuint64_t(d->length), cuuint64_t(d->batch)};
    const cuuint64_t strides[2] = {cuuint64_t(step) * es, cuuint64_t(batch) * es};
    const cuuint32_t box[3] = {cuuint32_t(tile_channels), cuuint32_t(kScanTile), 1};
    return one(map, 3, p, dims, strides, box);
  };
  auto states = [&](CUtensorMap* map, const void* p, int64_t batch, int64_t step, int64_t group) {
    const cuuint64_t dims[4] = {cuuint64_t(d->states), cuuint64_t(d->groups), cuuint64_t(d->length),
                                cuuint64_t(d->batch)};
    const cuuint64_t strides[3] = {cuuint64_t(group) * es, cuuint64_t(step) * es, cuuint64_t(batch) * es};
    const cuuint32_t box[4] = {cuuint32_t(pad), 1, cuuint32_t(kScanTile), 1};
    return one(map, 4, p, dims, strides, box);
  };
  // A box may not be larger than its tensor, and a tile may not reach into the next group's channels: what it
  // holds behind its own has to be zeros (the copy engine's, behind the last channel).
  if (d->channels < tile_channels || d->length < kScanTile || d->states < pad) return false;
  if (d->groups > 1 && (d->channels / d->groups) % tile_channels) return false;
  return act(&m->u, u, d->u_batch, d->u_step) && act(&m->delta, delta, d->delta_batch, d->delta_step) &&
         (!z || act(&m->z, z, d->z_batch, d->z_step)) && (!dy || act(&m->dy, dy, d->dy_batch, d->dy_step)) &&
         states(&m->B, B, d->B_batch, d->B_step, d->B_group) && states(&m->C, C, d->C_batch, d->C_step, d->C_group);
}

template <typename T, class Sh>
static int scan_forward_launch(const bst_scan_desc* d, ScanArgs a, cudaStream_t st) {
  a.col_tiles = (a.per_group + Sh::CT - 1) / Sh::CT;
  const int64_t blocks = int64_t(a.batch) * a.groups * a.col_tiles;
  if (blocks > INT_MAX) return fail(BST_ERR_UNSUPPORTED, "the scan needs more than 2^31 blocks");
  ScanMaps maps;
  if (a.mode == kCopyTiles && !scan_maps(d, Sh::CT, Sh::NP, a.u, a.delta, a.z, nullptr, a.B, a.C, &maps))
    a.mode = kCopyWords;
  constexpr int smem = int(sizeof(ForwardRaw<T, Sh>));
  auto* kernel = a.mode == kCopyTiles ? scan_forward_kernel<T, Sh, true> : scan_forward_kernel<T, Sh, false>;
  BST_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
  kernel<<<unsigned(blocks), 2 * Sh::NT, smem, st>>>(a, maps);
  return launched("scan_forward_kernel launch");
}

}  // namespace bst

using namespace bst;

extern "C" {

int bst_scan_workspace(const bst_scan_desc* d, int32_t what, int64_t* bytes) {
  clear_error();
  if (int rc = scan_check(d)) return rc;
  if (!bytes) return fail(BST_ERR_INVALID, "null output");
  if (what == BST_SCAN_BACKWARD) *bytes = scan_backward_workspace(d);
  else if (what == BST_SCAN_SAVED) *bytes = scan_saved_bytes(d);
  else return fail(BST_ERR_INVALID, "unknown workspace");
  return BST_OK;
}

int bst_scan_forward(const bst_scan_desc* d, const void* u, const void* delta, const float* A, const void* B,
                     const void* C, const float* D, const void* z, const float* delta_bias, const float* initial,
                     const int32_t* lengths, void* y, float* final_state, void* saved, void* stream) {
  clear_error();
  if (int rc = scan_check(d)) return rc;
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
  if (!aligned16(saved)) return fail(BST_ERR_INVALID, "the saved states must be aligned to 16 bytes");
  ScanArgs a = scan_args(d);
  a.u = u, a.delta = delta, a.A = A, a.B = B, a.C = C, a.D = D, a.z = z, a.dbias = delta_bias, a.init = initial;
  a.lengths = lengths, a.y = y, a.final_state = final_state, a.saved = static_cast<float*>(saved);
  const int64_t per = 16 / layer_elem_size(d->dtype);
  a.vec = aligned16(u) && aligned16(delta) && aligned16(z) && aligned16(y) &&
          (a.per_group | a.ub | a.us | a.db | a.ds | (z ? a.zb | a.zs : 0) | a.yb | a.ys) % per == 0;
  a.mode = scan_copy_mode(d, u, delta, z, nullptr, B, C);
  a.error = device_error_word();
  if (!a.error) return fail(BST_ERR_CUDA, "device error word unavailable");
  return with_type(d->dtype, [&](auto t) {
    using T = decltype(t);
    // Two channels per lane halve the shared-memory bytes and the sums' shuffles per recurrence; one channel, or one
    // with half of the states, doubles the warps each time, which pays while they are scarce.  By channel-state pairs
    // per scheduler of the GPU; with 16 states in bf16, 2 channels x 4 states | 1 x 4 | 1 x 2 per lane:
    // 4 x 2048 x 4096: 324 | 410 | 426 us, 1 x 4096 x 8192: 370 | 414 | 503, 1 x 4096 x 4096: 364 | 261 | 268,
    // 1 x 4096 x 1024: 361 | 256 | 174.
    const int64_t pairs = d->batch * d->channels * scan_pad(d->states) / (int64_t(sm_count()) * 4);
    switch (scan_pad(d->states)) {
      case 4: return scan_forward_launch<T, ScanShape<2, 2, 2, 2>>(d, a, st);
      case 8: return scan_forward_launch<T, ScanShape<4, 2, 2, 2>>(d, a, st);
      case 16:
        if (pairs >= 192) return scan_forward_launch<T, ScanShape<4, 2, 4, 4>>(d, a, st);
        if (pairs >= 64) return scan_forward_launch<T, ScanShape<4, 1, 4, 4>>(d, a, st);
        return scan_forward_launch<T, ScanShape<2, 1, 8, 4>>(d, a, st);
      case 32:
        if (pairs >= 192) return scan_forward_launch<T, ScanShape<4, 2, 8, 4>>(d, a, st);
        return scan_forward_launch<T, ScanShape<4, 1, 8, 4>>(d, a, st);
      default: return scan_forward_launch<T, ScanShape<4, 2, 16, 4>>(d, a, st);
    }
  });
}

}  // extern "C"
