// The gated scan backward (tgdn_scan.cuh): the whole way, the tiles' reverse maps, and the gradients from the mu between the tiles.
#include "tgdn_scan.cuh"

namespace tgdn {

// Blocks an SM that the registers are shared among.  Pairs of channels in packed rows get one: at two, 128 registers a thread, they would spill 300
// bytes and more, and took longer even where there are two blocks for each SM (bf16, one row of 8192 x 16384: 467 -> 445 us; of 16384 x 8192, 128
// blocks: 775 -> 396 us).  So do pairs of more than four bytes in x and g, whose stages leave no room for a second block; the maps alone fit twice.
// Single channels of 16-bit rows fit twice with few spills or none (f32 gates, 8 x 4096 x 1001: 189 -> 140 us; packed 16384 x 8001: 936 -> 734);
// f32 rows keep their prefetch at one (8 x 4096 x 1001: 178 -> 150 us).
constexpr int bwd_per_sm(int x_bytes, int g_bytes, bool ring, bool packed, int way) {
  return way == SCAN_MAPS || (x_bytes == 2 && (!ring || (g_bytes == 2 && !packed))) ? 2 : 1;
}

// WIDE: once more over the block's tiles, with factors out of range.
template <typename TX, typename TG, bool RING, bool PACKED, int WAY, bool WIDE, int VEC>
__device__ __forceinline__ void scan_bwd_walk(const ScanParams& p, const Place<VEC>& at, SharedMaps<VEC, PACKED>* maps, Ring<TX, TG, WAY != SCAN_MAPS, true>& ring) {
  constexpr bool STATES = WAY != SCAN_MAPS;      // (the reverse maps need neither x nor h)
  using MapT = Map<VEC, PACKED>;
  using RingT = Ring<TX, TG, STATES, true>;
  const int lane = at.lane, warp = at.warp, c0 = at.c0;
  const bool active = at.active, asks = RING && threadIdx.x == 0;
  const int64_t xb = at.b * p.x.sb + (active ? c0 : 0), gb = at.b * p.g.sb + (active ? c0 : 0), hb = at.b * p.dh.sb + (active ? c0 : 0);
  // mu behind the tile, the same in every warp
  Lanes<VEC> carry = load_f32<VEC>(p.dfinal + at.state, WAY == SCAN_WHOLE && !PACKED && p.dfinal && active);
  if (WAY == SCAN_FINISH) carry = load_f32<VEC>(p.mu + at.at_tile(p, at.hi - 1), active);

  RawRows<TX, VEC> xr, hr;
  RawRows<TG, VEC> gr;
  auto request = [&](int t0) {
    if constexpr (!RING) {
      if constexpr (STATES) request_rows<TX>(p.x, xb, t0, p.T, xr);
      request_rows<TG>(p.g, gb, t0, p.T, gr);
      request_rows<TX>(p.dh, hb, t0, p.T, hr);
    }
  };
  auto saved = [&](int tile) { return load_f32<VEC>(p.carry + at.at_tile(p, tile), STATES && active && tile >= at.lo); };   // the state before a tile
  if (asks)
    for (int n = 0; n < p.stages && at.hi - 1 - n >= at.lo; ++n) ring.request((at.hi - 1 - n) * SCAN_TILE);
  if (!WIDE) request((at.hi - 1) * SCAN_TILE + warp * SCAN_ROWS);   // (the second walk has no registers for rows ahead)
  int code = row_code<PACKED>(p, (at.hi - 1) * SCAN_TILE + warp * SCAN_ROWS, lane);
  Lanes<VEC> next_h = saved(at.hi - 1);
  for (int tile = at.hi - 1; tile >= at.lo; --tile) {
    const int t0 = tile * SCAN_TILE + warp * SCAN_ROWS, buf = tile & 1;
    const bool more = tile > at.lo;
    Lanes<VEC> a[SCAN_ROWS], x[SCAN_ROWS], dh[SCAN_ROWS], next_carry;
    if (RING) {
      const uint8_t* here = ring.wait();
      if constexpr (STATES) take_rows<TX, VEC>(here + RingT::X_AT, warp, lane, xr);
      take_rows<TG, VEC>(here, warp, lane, gr);
      take_rows<TX, VEC>(here + RingT::DH_AT, warp, lane, hr);
      ring.advance();
    }
    if (WIDE) request(t0);
    if constexpr (STATES) unpack_rows<TX, VEC>(xr, x);
    unpack_rows<TG, VEC>(gr, a);
    unpack_rows<TX, VEC>(hr, dh);
    if (!WIDE && more) request(t0 - SCAN_TILE);
    const RowDocs docs = row_docs<PACKED>(p, t0, code);
    const bool cuts = PACKED && docs.any();
    Lanes<VEC> h = next_h;
    if (more) {
      code = row_code<PACKED>(p, t0 - SCAN_TILE, lane);
      next_h = saved(tile - 1);
    }
    if (WAY == SCAN_FINISH) next_carry = load_f32<VEC>(p.mu + at.at_tile(p, tile - 1), more && active);
    decays<VEC>(a);
    MapT run = MapT::identity(), back = run;
    if (cuts) {
      if (STATES && p.initial) bring_states<VEC>(p, docs, c0, active, a, x);
      if (p.dfinal) {                            // the gradient of a final state comes in with its document's last token
#pragma unroll
        for (int r = 0; r < SCAN_ROWS; ++r)
          if (docs.ends_at(r)) {
            const int doc = docs.closed(r);
            dh[r] = add(dh[r], load_f32<VEC>(p.dfinal + static_cast<int64_t>(doc) * p.D + c0, active && doc >= 0));
          }
      }
      run.cut = docs.starts != 0;
      back.cut = docs.ends != 0;
      if constexpr (STATES) run_forward<true, VEC>(docs, a, x, run.A, run.H);
      run_reverse<true, VEC>(docs, a, dh, back.H);
    } else {
      if constexpr (STATES) run_forward<false, VEC>(docs, a, x, run.A, run.H);
      run_reverse<false, VEC>(docs, a, dh, back.H);
    }
    if constexpr (!STATES)
#pragma unroll
      for (int r = 0; r < SCAN_ROWS; ++r) run.A = mul(run.A, a[r]);
    if (WIDE) run.widen(a);
    else if (!run.moderate()) ring.control->wide = 1;
    back.A = run.A;
    maps[0].put(buf, warp, lane, back);
    if constexpr (STATES) maps[1].put(buf, warp, lane, run);
    const bool tile_cuts = maps_written<PACKED>((run.cut | back.cut) != 0);
    if (asks && tile - p.stages >= at.lo && !ring.given_up()) ring.request((tile - p.stages) * SCAN_TILE);

    if constexpr (WAY == SCAN_MAPS) {
      if (warp == tile % SCAN_WARPS)
        by_cuts<PACKED>(tile_cuts, [&](auto in_tile) {
          constexpr bool CUTS = decltype(in_tile)::value;
          Map<VEC, CUTS> whole = Map<VEC, CUTS>::identity();
          if constexpr (WIDE) {
            whole = compose_wide<true, VEC, CUTS>(maps[0], buf, lane, SCAN_WARPS - 1, -1, SCAN_WARPS, carry, carry);
          } else {
            compose<true>(whole, maps[0], buf, lane, SCAN_WARPS - 1, -1);
          }
          leave_map(p, at, tile, whole);
        });
      continue;
    } else {
      by_cuts<PACKED>(tile_cuts, [&](auto in_tile) {
        constexpr bool CUTS = decltype(in_tile)::value;
        if constexpr (WIDE) {
          const Lanes<VEC> first = h;
          compose_wide<false, VEC, CUTS>(maps[1], buf, lane, 0, warp, warp, first, h);
        } else {
          Map<VEC, CUTS> before = Map<VEC, CUTS>::identity();
          compose<false>(before, maps[1], buf, lane, 0, warp);
          before.apply(h);
        }
      });
      if (cuts) {                                // x becomes the state before its row
#pragma unroll
        for (int r = 0; r < SCAN_ROWS; ++r) {
          Lanes<VEC> last = h;
          if (docs.starts_at(r))
            last = p.initial ? load_f32<VEC>(p.initial + static_cast<int64_t>(docs.opened(r)) * p.D + c0, active) : all<VEC>(0.f);
          h = docs.starts_at(r) ? x[r] : fma(a[r], h, x[r]);
          x[r] = last;
        }
      } else {
#pragma unroll
        for (int r = 0; r < SCAN_ROWS; ++r) {
          const Lanes<VEC> last = h;
          h = fma(a[r], h, x[r]);
          x[r] = last;
        }
      }
      Lanes<VEC> mu = carry;
      by_cuts<PACKED>(tile_cuts, [&](auto in_tile) {
        constexpr bool CUTS = decltype(in_tile)::value;
        Map<VEC, CUTS> whole = Map<VEC, CUTS>::identity();
        if constexpr (WIDE) {
          whole = compose_wide<true, VEC, CUTS>(maps[0], buf, lane, SCAN_WARPS - 1, WAY == SCAN_WHOLE ? -1 : warp, warp, carry, mu);
          if (WAY == SCAN_WHOLE) whole.apply_wide(carry);
        } else {
          compose<true>(whole, maps[0], buf, lane, SCAN_WARPS - 1, warp);
          whole.apply(mu);
          if (WAY == SCAN_WHOLE) {
            compose<true>(whole, maps[0], buf, lane, warp, -1);
            whole.apply(carry);
          }
        }
      });
      if (WAY == SCAN_FINISH) carry = next_carry;

      const int64_t row = (static_cast<int64_t>(at.b) * p.T + t0) * p.D + c0;
      TX* dx = static_cast<TX*>(p.dx) + row;
      TG* dg = static_cast<TG*>(p.dg) + row;
      const int rows = active ? p.T - t0 : 0, stride = opaque(p.D);
      by_cuts<PACKED>(cuts, [&](auto in_rows) {
        constexpr bool CUTS = decltype(in_rows)::value;
        Lanes<VEC> lam = CUTS && docs.ends_at(SCAN_ROWS - 1) ? dh[SCAN_ROWS - 1] : add(dh[SCAN_ROWS - 1], mu);
#pragma unroll
        for (int r = SCAN_ROWS - 1; r >= 0; --r) {
          if (r < SCAN_ROWS - 1) lam = CUTS && docs.ends_at(r) ? dh[r] : fma(a[r + 1], lam, dh[r]);
          mu = mul(a[r], lam);
          const Lanes<VEC> d = mul(mu, x[r]);
          if (r < rows) {
            store_f32_as<TX, VEC>(row_of(dx, r, stride), lam.v);
            store_f32_as<TG, VEC>(row_of(dg, r, stride), d.v);
          }
          if (CUTS && p.dinitial && docs.starts_at(r)) {
            const int doc = docs.opened(r);
            if (active) store_f32<VEC>(p.dinitial + static_cast<int64_t>(doc) * p.D + c0, mu);
          }
        }
      });
    }
  }
  if (WAY == SCAN_WHOLE && !PACKED && p.dinitial && warp == 0 && active) store_f32<VEC>(p.dinitial + at.state, carry);
  if (asks && ring.given_up()) ring.drain();
}
// A function of its own, so that the plain walk keeps its registers.
template <typename TX, typename TG, bool RING, bool PACKED, int WAY, int VEC>
__device__ __noinline__ void scan_bwd_again(const ScanParams& p, SharedMaps<VEC, PACKED>* maps, Ring<TX, TG, WAY != SCAN_MAPS, true> ring) {
  const Place<VEC> at(p, WAY == SCAN_FINISH);
  scan_bwd_walk<TX, TG, RING, PACKED, WAY, true, VEC>(p, at, maps, ring);
}

template <typename TX, typename TG, bool RING, bool PACKED, int WAY>
__global__ void __launch_bounds__(32 * SCAN_WARPS, bwd_per_sm(sizeof(TX), sizeof(TG), RING, PACKED, WAY))
scan_bwd_kernel(const __grid_constant__ ScanMaps tensors, const __grid_constant__ ScanParams p) {
  constexpr int VEC = RING ? 2 : 1;
  constexpr bool STATES = WAY != SCAN_MAPS;
  extern __shared__ __align__(128) uint8_t dynamic[];
  __shared__ SharedMaps<VEC, PACKED> maps[STATES ? 2 : 1];     // reverse, forward
  __shared__ RingControl control;
  const Place<VEC> at(p, WAY == SCAN_FINISH);
  Ring<TX, TG, STATES, true> ring(tensors, dynamic, &control, p.status, at.slice0, at.b, RING ? p.stages : 0);
  scan_bwd_walk<TX, TG, RING, PACKED, WAY, false, VEC>(p, at, maps, ring);
  __syncthreads();
  if (control.wide && !ring.given_up()) scan_bwd_again<TX, TG, RING, PACKED, WAY, VEC>(p, maps, ring);   // (a block that gave up asks for nothing more)
}

}  // namespace tgdn

using namespace tgdn;

namespace {
template <int WAY>
struct Backward {
  template <typename TX, typename TG, bool RING, bool PACKED>
  static int go(ScanParams p, cudaStream_t s) {
    static bool configured[64] = {false};
    constexpr int VEC = RING ? 2 : 1, fixed = (WAY == SCAN_MAPS ? 1 : 2) * static_cast<int>(sizeof(SharedMaps<VEC, PACKED>)) + 256;
    p.slices = (p.D + 32 * VEC - 1) / (32 * VEC);
    return scan_launch<RING, TX, TG, WAY != SCAN_MAPS, true, bwd_per_sm(sizeof(TX), sizeof(TG), RING, PACKED, WAY)>(scan_bwd_kernel<TX, TG, RING, PACKED, WAY>, configured, fixed, p, s);
  }
};
}  // namespace

int tgdn_scan_launch_bwd(const ScanParams& p, int xt, int gt, bool pieces, ScanWay way, cudaStream_t s) {
  if (way == SCAN_WHOLE) return scan_launch_any<Backward<SCAN_WHOLE>>(p, xt, gt, pieces, s);
  return way == SCAN_MAPS ? scan_launch_any<Backward<SCAN_MAPS>>(p, xt, gt, pieces, s) : scan_launch_any<Backward<SCAN_FINISH>>(p, xt, gt, pieces, s);
}
