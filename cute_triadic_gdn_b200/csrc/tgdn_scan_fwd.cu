// The gated scan forward (tgdn_scan.cuh): the whole way, the tiles' maps, and the outputs from the states between the tiles.
#include "tgdn_scan.cuh"

namespace tgdn {

// Blocks an SM that the registers are shared among: two of 128 a thread with 16-bit rows, none of which spills.
constexpr int fwd_per_sm(int x_bytes) { return x_bytes == 2 ? 2 : 1; }

// RING: pairs of channels, tiles by the copy engine (rows of whole 16-byte pieces).  Otherwise single channels by plain loads of any
// alignment, the next tile in registers.
// WIDE: once more over the block's tiles, with factors out of range.
template <typename TX, typename TG, bool RING, bool PACKED, int WAY, bool WIDE, int VEC>
__device__ __forceinline__ void scan_fwd_walk(const ScanParams& p, const Place<VEC>& at, SharedMaps<VEC, PACKED>& maps, Ring<TX, TG, true, false>& ring) {
  using MapT = Map<VEC, PACKED>;
  using RingT = Ring<TX, TG, true, false>;
  const int lane = at.lane, warp = at.warp, c0 = at.c0;
  const bool active = at.active, asks = RING && threadIdx.x == 0;
  const int64_t xb = at.b * p.x.sb + (active ? c0 : 0), gb = at.b * p.g.sb + (active ? c0 : 0);
  // the state before the tile, the same in every warp
  Lanes<VEC> carry = load_f32<VEC>(p.initial + at.state, WAY == SCAN_WHOLE && !PACKED && p.initial && active);
  if (WAY == SCAN_FINISH) carry = load_f32<VEC>(p.carry + at.at_tile(p, at.lo), active);

  RawRows<TX, VEC> xr;
  RawRows<TG, VEC> gr;
  if (asks)
    for (int n = 0; n < p.stages && at.lo + n < at.hi; ++n) ring.request((at.lo + n) * SCAN_TILE);
  const auto request = [&](int t0) {
    if constexpr (!RING) {
      request_rows<TX>(p.x, xb, t0, p.T, xr);
      request_rows<TG>(p.g, gb, t0, p.T, gr);
    }
  };
  if (!WIDE) request(at.lo * SCAN_TILE + warp * SCAN_ROWS);           // (the second walk has no registers for rows ahead)
  int code = row_code<PACKED>(p, at.lo * SCAN_TILE + warp * SCAN_ROWS, lane);
  for (int tile = at.lo; tile < at.hi; ++tile) {
    const int t0 = tile * SCAN_TILE + warp * SCAN_ROWS, buf = tile & 1;
    const bool more = tile + 1 < at.hi;
    Lanes<VEC> a[SCAN_ROWS], x[SCAN_ROWS], next_carry;
    if (RING) {
      const uint8_t* here = ring.wait();
      take_rows<TX, VEC>(here + RingT::X_AT, warp, lane, xr);
      take_rows<TG, VEC>(here, warp, lane, gr);
      ring.advance();
    }
    if (WIDE) request(t0);
    unpack_rows<TX, VEC>(xr, x);
    unpack_rows<TG, VEC>(gr, a);
    if (!WIDE && more) request(t0 + SCAN_TILE);
    const RowDocs docs = row_docs<PACKED>(p, t0, code);
    if (more) code = row_code<PACKED>(p, t0 + SCAN_TILE, lane);
    if (WAY == SCAN_FINISH) next_carry = load_f32<VEC>(p.carry + at.at_tile(p, tile + 1), more && active);
    const bool cuts = PACKED && docs.any();
    decays<VEC>(a);
    MapT run = MapT::identity();
    if (cuts) {
      if (p.initial) bring_states<VEC>(p, docs, c0, active, a, x);
      run.cut = docs.starts != 0;
      run_forward<true, VEC>(docs, a, x, run.A, run.H);
    } else {
      run_forward<false, VEC>(docs, a, x, run.A, run.H);
    }
    if (WIDE) run.widen(a);
    else if (!run.moderate()) ring.control->wide = 1;
    maps.put(buf, warp, lane, run);
    const bool tile_cuts = maps_written<PACKED>(run.cut != 0);
    if (asks && tile + p.stages < at.hi && !ring.given_up()) ring.request((tile + p.stages) * SCAN_TILE);   // every warp has its rows

    if (WAY == SCAN_MAPS) {
      if (warp == tile % SCAN_WARPS)
        by_cuts<PACKED>(tile_cuts, [&](auto in_tile) {
          constexpr bool CUTS = decltype(in_tile)::value;
          Map<VEC, CUTS> whole = Map<VEC, CUTS>::identity();
          if constexpr (WIDE) {
            whole = compose_wide<false, VEC, CUTS>(maps, buf, lane, 0, SCAN_WARPS, -1, carry, carry);
          } else {
            AllMaps<VEC, CUTS>(maps, buf, lane).compose(whole, 0, SCAN_WARPS);
          }
          leave_map(p, at, tile, whole);
        });
      continue;
    }
    Lanes<VEC> mine = carry;
    by_cuts<PACKED>(tile_cuts, [&](auto in_tile) {
      // the maps of the warps before this one, and of all of the block; then the state before the warp's rows
      constexpr bool CUTS = decltype(in_tile)::value;
      Map<VEC, CUTS> whole = Map<VEC, CUTS>::identity();
      if (WAY == SCAN_WHOLE && p.carry && warp == 0 && active) store_f32<VEC>(p.carry + at.at_tile(p, tile), carry);
      const auto go = [&](auto composed) {
        composed(whole, 0, warp);
        whole.apply(mine);
        if (WAY == SCAN_WHOLE) {
          composed(whole, warp, SCAN_WARPS);
          whole.apply(carry);
        }
      };
      if constexpr (WIDE) {
        whole = compose_wide<false, VEC, CUTS>(maps, buf, lane, 0, WAY == SCAN_WHOLE ? SCAN_WARPS : warp, warp, carry, mine);
        if (WAY == SCAN_WHOLE) whole.apply_wide(carry);
      } else if constexpr (CUTS) {
        go([&](auto& to, int lo, int hi) { compose<false>(to, maps, buf, lane, lo, hi); });
      } else {
        const AllMaps<VEC, CUTS> tile_maps(maps, buf, lane);
        go([&](auto& to, int lo, int hi) { tile_maps.compose(to, lo, hi); });
      }
    });
    if (WAY == SCAN_FINISH) carry = next_carry;

    TX* out = static_cast<TX*>(p.h) + (static_cast<int64_t>(at.b) * p.T + t0) * p.D + c0;
    const int rows = active ? p.T - t0 : 0, stride = opaque(p.D);
    if (cuts) {
#pragma unroll
      for (int r = 0; r < SCAN_ROWS; ++r) {
        mine = docs.starts_at(r) ? x[r] : fma(a[r], mine, x[r]);
        if (r < rows) store_f32_as<TX, VEC>(row_of(out, r, stride), mine.v);
        if (p.final_state && docs.ends_at(r)) {
          const int doc = docs.closed(r);
          if (active && doc >= 0) store_f32<VEC>(p.final_state + static_cast<int64_t>(doc) * p.D + c0, mine);
        }
      }
    } else {
#pragma unroll
      for (int r = 0; r < SCAN_ROWS; ++r) {
        mine = fma(a[r], mine, x[r]);
        if (r < rows) store_f32_as<TX, VEC>(row_of(out, r, stride), mine.v);
      }
    }
  }
  // Rows past T are identity maps (a = 1, x = 0), so the state behind the last tile is the one after the last token.
  if (WAY == SCAN_WHOLE && !PACKED && p.final_state && warp == 0 && active) store_f32<VEC>(p.final_state + at.state, carry);
  if (asks && ring.given_up()) ring.drain();
}
// A function of its own, so that the plain walk keeps its registers.
template <typename TX, typename TG, bool RING, bool PACKED, int WAY, int VEC>
__device__ __noinline__ void scan_fwd_again(const ScanParams& p, SharedMaps<VEC, PACKED>& maps, Ring<TX, TG, true, false> ring) {
  const Place<VEC> at(p, WAY == SCAN_FINISH);
  scan_fwd_walk<TX, TG, RING, PACKED, WAY, true, VEC>(p, at, maps, ring);
}

template <typename TX, typename TG, bool RING, bool PACKED, int WAY>
__global__ void __launch_bounds__(32 * SCAN_WARPS, fwd_per_sm(sizeof(TX)))
scan_fwd_kernel(const __grid_constant__ ScanMaps tensors, const __grid_constant__ ScanParams p) {
  constexpr int VEC = RING ? 2 : 1;
  extern __shared__ __align__(128) uint8_t dynamic[];
  __shared__ SharedMaps<VEC, PACKED> maps;
  __shared__ RingControl control;
  const Place<VEC> at(p, WAY == SCAN_FINISH);
  Ring<TX, TG, true, false> ring(tensors, dynamic, &control, p.status, at.slice0, at.b, RING ? p.stages : 0);
  scan_fwd_walk<TX, TG, RING, PACKED, WAY, false, VEC>(p, at, maps, ring);
  __syncthreads();
  if (control.wide && !ring.given_up()) scan_fwd_again<TX, TG, RING, PACKED, WAY, VEC>(p, maps, ring);   // (a block that gave up asks for nothing more)
}

}  // namespace tgdn

using namespace tgdn;

namespace {
template <int WAY>
struct Forward {
  template <typename TX, typename TG, bool RING, bool PACKED>
  static int go(ScanParams p, cudaStream_t s) {
    static bool configured[64] = {false};
    constexpr int VEC = RING ? 2 : 1, fixed = static_cast<int>(sizeof(SharedMaps<VEC, PACKED>)) + 256;
    p.slices = (p.D + 32 * VEC - 1) / (32 * VEC);
    return scan_launch<RING, TX, TG, true, false, fwd_per_sm(sizeof(TX))>(scan_fwd_kernel<TX, TG, RING, PACKED, WAY>, configured, fixed, p, s);
  }
};
}  // namespace

int tgdn_scan_launch_fwd(const ScanParams& p, int xt, int gt, bool pieces, ScanWay way, cudaStream_t s) {
  if (way == SCAN_WHOLE) return scan_launch_any<Forward<SCAN_WHOLE>>(p, xt, gt, pieces, s);
  return way == SCAN_MAPS ? scan_launch_any<Forward<SCAN_MAPS>>(p, xt, gt, pieces, s) : scan_launch_any<Forward<SCAN_FINISH>>(p, xt, gt, pieces, s);
}
