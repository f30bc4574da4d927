// Gated linear recurrence per channel:  h[t] = exp(g[t]) h[t-1] + x[t]  over (B, T, D), forward, backward and one token.
//
// With a = exp(g) a run of rows maps the state c before it to the state behind it by c -> A c + H, A the product of its a and H its own
// result from zero; such maps compose, so the time axis is cut into runs that are walked at the same time.  The gradient runs the other
// way: with lam[t] = dL/dh[t] and mu[t] = a[t] lam[t],
//     lam[t] = dh[t] + mu[t+1],   dx[t] = lam[t],   dg[t] = mu[t] h[t-1],   dinitial = mu[first],
// and a run maps the mu behind it to the mu before it by mu -> A mu + M with the same A.
//
// A warp holds 16 rows of 32 * VEC channels in registers (a lane VEC channels, a row of the warp one coalesced access), a block of eight
// warps a tile of 128 rows; tiles follow one another along time with the state in registers.  Every input is read once and every output
// written once: 6 bytes an element forward and 10 backward in 16 bits, which is the bound (HBM).  The backward forms h again from x and
// the f32 state at the start of every tile, which the forward leaves (4 bytes per 128 rows and channel): the output in 16 bits would put
// its rounding into dg, and would have to be read in the place of x.
//
// Sums, products and states are f32.  Maps are composed in an order given by the tile alone, so a sequence's results do not depend on
// what runs beside it.
#include "tgdn_common.cuh"
#include "tgdn_host.h"
#include "tgdn_rows.cuh"

namespace tgdn {

constexpr int SCAN_ROWS = 16;                    // rows a warp holds
constexpr int SCAN_WARPS = 8;
constexpr int SCAN_TILE = SCAN_ROWS * SCAN_WARPS;
static_assert(SCAN_TILE == TGDN_SCAN_TILE, "rows between two saved states");

struct ScanIn {
  const void* p;
  int64_t sb, st;                                // elements from one batch row, and from one token, to the next
};

struct ScanParams {
  ScanIn x, g, dh;
  const int32_t* map;                            // packed: document + 1 at its first token, 0 elsewhere
  const float* initial;                          // (sequences, D) or nullptr
  const float* dfinal;
  void* h;                                       // forward: output;  backward: unused
  float* final_state;
  float* carry;                                  // (B, tiles, D): the state before every tile
  void* dx;
  void* dg;
  float* dinitial;
  int B, T, D, n_docs, slices, tiles;
};

// exp(g).  Near zero as 1 + (g + g^2/2 + ...): the sum is rounded once, to nearest, while the hardware's power of two errs by up to two
// units to one side, and such errors add up over as many tokens as the state remembers (a thousand tokens at g = -1e-3: 2e-5 where
// roundings to nearest leave 1e-6).  Beyond 1/8 a state remembers eight tokens at most and the power of two is good enough.  The series
// to the fifth power is 2^-28 off at 1/8.
__device__ __forceinline__ float decay(float g) {
  float s = fmaf(g, 1.f / 120.f, 1.f / 24.f);
  s = fmaf(g, s, 1.f / 6.f);
  s = fmaf(g, s, 0.5f);
  s = fmaf(g, s, 1.f);
  s = fmaf(g, s, 1.f);
  return fabsf(g) < 0.125f ? s : exp2f(g * 1.4426950408889634f);
}

template <int VEC>
struct Channels {
  float v[VEC];
};

// What a warp knows about the documents of its rows: bit r of `starts`, row r opens a document (whose number + 1 lane r holds); bit r of
// `ends`, it closes one.
struct RowDocs {
  uint32_t starts, ends;
  int code;
  __device__ int opened(int r) const { return __shfl_sync(0xffffffffu, code, r) - 1; }
  // The document before the one that opens at the next row; -1 where offsets that do not start at 0 leave none.
  __device__ int closed(int r) const { return __shfl_sync(0xffffffffu, code, r + 1) - 2; }
};

template <bool PACKED>
__device__ __forceinline__ RowDocs row_docs(const ScanParams& p, int t0, int lane) {
  RowDocs d{0u, 0u, 0};
  if constexpr (PACKED) {
    const int t = t0 + lane;
    if (lane <= SCAN_ROWS) d.code = t < p.T ? p.map[t] : t == p.T ? p.n_docs + 1 : 0;
    const uint32_t b = __ballot_sync(0xffffffffu, d.code != 0);
    d.starts = b & ((1u << SCAN_ROWS) - 1);
    if (t0 + SCAN_ROWS > p.T && t0 <= p.T) d.starts &= (1u << (p.T - t0)) - 1;
    d.ends = (b >> 1) & ((1u << SCAN_ROWS) - 1);
  }
  return d;
}

template <typename T, int VEC>
__device__ __forceinline__ void load_rows(const ScanIn& in, int64_t base, int t0, int T_, bool active, float (&out)[SCAN_ROWS][VEC]) {
  Pack<T, VEC> raw[SCAN_ROWS];
  const T* p = static_cast<const T*>(in.p) + base;
#pragma unroll
  for (int r = 0; r < SCAN_ROWS; ++r)
    raw[r] = active && t0 + r < T_ ? load_pack<T, VEC>(p + (t0 + r) * in.st) : zero_pack<T, VEC>();
#pragma unroll
  for (int r = 0; r < SCAN_ROWS; ++r)
#pragma unroll
    for (int i = 0; i < VEC; ++i) out[r][i] = to_f32(raw[r].v[i]);
}

// The maps of a block's warps, double-buffered: a tile's are written while slower warps still read the last one's.
template <int VEC, int MAPS>
struct alignas(16) WarpMaps {
  float v[2][MAPS][SCAN_WARPS][32 * VEC];
  int cut[2][2][SCAN_WARPS];                     // [buffer][forward, reverse][warp]: no state passes through
};

template <int VEC>
__device__ __forceinline__ Channels<VEC> read_map(const float* row, int lane) {
  Channels<VEC> c;
#pragma unroll
  for (int i = 0; i < VEC; ++i) c.v[i] = row[lane * VEC + i];
  return c;
}
template <int VEC>
__device__ __forceinline__ void write_map(float* row, int lane, const float (&v)[VEC]) {
#pragma unroll
  for (int i = 0; i < VEC; ++i) row[lane * VEC + i] = v[i];
}

template <typename TX, typename TG, int VEC, bool PACKED>
__global__ void __launch_bounds__(32 * SCAN_WARPS)
scan_fwd_kernel(ScanParams p) {
  __shared__ WarpMaps<VEC, 2> maps;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int slice = blockIdx.x % p.slices, b = blockIdx.x / p.slices;
  const int c0 = (slice * 32 + lane) * VEC;
  const bool active = c0 < p.D;
  const int64_t xb = b * p.x.sb + c0, gb = b * p.g.sb + c0;
  float carry[VEC];                              // the state before the tile, the same in every warp
#pragma unroll
  for (int i = 0; i < VEC; ++i)
    carry[i] = !PACKED && p.initial && active ? p.initial[static_cast<int64_t>(b) * p.D + c0 + i] : 0.f;

  for (int tile = 0; tile < p.tiles; ++tile) {
    const int t0 = tile * SCAN_TILE + warp * SCAN_ROWS, buf = tile & 1;
    float a[SCAN_ROWS][VEC], x[SCAN_ROWS][VEC];
    load_rows<TX, VEC>(p.x, xb, t0, p.T, active, x);
    load_rows<TG, VEC>(p.g, gb, t0, p.T, active, a);
    const RowDocs docs = row_docs<PACKED>(p, t0, lane);
    float A[VEC], H[VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) A[i] = 1.f, H[i] = 0.f;
#pragma unroll
    for (int r = 0; r < SCAN_ROWS; ++r) {
      const bool starts = PACKED && (docs.starts >> r & 1);
#pragma unroll
      for (int i = 0; i < VEC; ++i) a[r][i] = decay(a[r][i]);
      if (PACKED && starts && p.initial) {       // the document's own state comes in with its first token
        const int64_t at = static_cast<int64_t>(docs.opened(r)) * p.D + c0;
#pragma unroll
        for (int i = 0; i < VEC; ++i) x[r][i] = fmaf(a[r][i], active ? p.initial[at + i] : 0.f, x[r][i]);
      }
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        H[i] = starts ? x[r][i] : fmaf(a[r][i], H[i], x[r][i]);
        A[i] *= a[r][i];
      }
    }
    write_map<VEC>(maps.v[buf][0][warp], lane, A);
    write_map<VEC>(maps.v[buf][1][warp], lane, H);
    if (PACKED && lane == 0) maps.cut[buf][0][warp] = docs.starts != 0;
    __syncthreads();

    // the map of the warps before this one, then of all, each applied to the state before the tile
    float mine[VEC], pa[VEC], ph[VEC];
    bool cut = false;
#pragma unroll
    for (int i = 0; i < VEC; ++i) pa[i] = 1.f, ph[i] = 0.f, mine[i] = carry[i];
    if (p.carry && warp == 0 && active) {
      float* at = p.carry + (static_cast<int64_t>(b) * p.tiles + tile) * p.D + c0;
#pragma unroll
      for (int i = 0; i < VEC; ++i) at[i] = carry[i];
    }
#pragma unroll
    for (int w = 0; w < SCAN_WARPS; ++w) {
      const Channels<VEC> wa = read_map<VEC>(maps.v[buf][0][w], lane), wh = read_map<VEC>(maps.v[buf][1][w], lane);
      const bool wcut = PACKED && maps.cut[buf][0][w];
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        if (w == warp) mine[i] = cut ? ph[i] : fmaf(pa[i], carry[i], ph[i]);
        ph[i] = wcut ? wh.v[i] : fmaf(wa.v[i], ph[i], wh.v[i]);
        pa[i] *= wa.v[i];
      }
      cut = cut || wcut;
    }
#pragma unroll
    for (int i = 0; i < VEC; ++i) carry[i] = cut ? ph[i] : fmaf(pa[i], carry[i], ph[i]);

    TX* out = static_cast<TX*>(p.h) + (static_cast<int64_t>(b) * p.T + t0) * p.D + c0;
#pragma unroll
    for (int r = 0; r < SCAN_ROWS; ++r) {
#pragma unroll
      for (int i = 0; i < VEC; ++i) mine[i] = PACKED && (docs.starts >> r & 1) ? x[r][i] : fmaf(a[r][i], mine[i], x[r][i]);
      if (active && t0 + r < p.T) store_pack<TX, VEC>(out + static_cast<int64_t>(r) * p.D, mine);
      if (PACKED && p.final_state && (docs.ends >> r & 1)) {
        const int doc = docs.closed(r);
        if (active && doc >= 0)
#pragma unroll
          for (int i = 0; i < VEC; ++i) p.final_state[static_cast<int64_t>(doc) * p.D + c0 + i] = mine[i];
      }
    }
  }
  // Rows past T are identity maps (a = 1, x = 0), so the state behind the last tile is the one after the last token.
  if (!PACKED && p.final_state && warp == 0 && active)
#pragma unroll
    for (int i = 0; i < VEC; ++i) p.final_state[static_cast<int64_t>(b) * p.D + c0 + i] = carry[i];
}

template <typename TX, typename TG, int VEC, bool PACKED>
__global__ void __launch_bounds__(32 * SCAN_WARPS)
scan_bwd_kernel(ScanParams p) {
  __shared__ WarpMaps<VEC, 3> maps;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int slice = blockIdx.x % p.slices, b = blockIdx.x / p.slices;
  const int c0 = (slice * 32 + lane) * VEC;
  const bool active = c0 < p.D;
  const int64_t xb = b * p.x.sb + c0, gb = b * p.g.sb + c0, hb = b * p.dh.sb + c0;
  float carry[VEC];                              // mu behind the tile, the same in every warp
#pragma unroll
  for (int i = 0; i < VEC; ++i) carry[i] = !PACKED && p.dfinal && active ? p.dfinal[static_cast<int64_t>(b) * p.D + c0 + i] : 0.f;

  for (int tile = p.tiles - 1; tile >= 0; --tile) {
    const int t0 = tile * SCAN_TILE + warp * SCAN_ROWS, buf = tile & 1;
    float a[SCAN_ROWS][VEC], x[SCAN_ROWS][VEC], dh[SCAN_ROWS][VEC];
    load_rows<TX, VEC>(p.x, xb, t0, p.T, active, x);
    load_rows<TG, VEC>(p.g, gb, t0, p.T, active, a);
    load_rows<TX, VEC>(p.dh, hb, t0, p.T, active, dh);
    const RowDocs docs = row_docs<PACKED>(p, t0, lane);
    float h[VEC];                                // the state before the tile
#pragma unroll
    for (int i = 0; i < VEC; ++i) h[i] = active ? p.carry[(static_cast<int64_t>(b) * p.tiles + tile) * p.D + c0 + i] : 0.f;
    float A[VEC], H[VEC], M[VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) A[i] = 1.f, H[i] = 0.f, M[i] = 0.f;
#pragma unroll
    for (int r = 0; r < SCAN_ROWS; ++r) {
      const bool starts = PACKED && (docs.starts >> r & 1);
#pragma unroll
      for (int i = 0; i < VEC; ++i) a[r][i] = decay(a[r][i]);
      if (PACKED && starts && p.initial) {
        const int64_t at = static_cast<int64_t>(docs.opened(r)) * p.D + c0;
#pragma unroll
        for (int i = 0; i < VEC; ++i) x[r][i] = fmaf(a[r][i], active ? p.initial[at + i] : 0.f, x[r][i]);
      }
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        H[i] = starts ? x[r][i] : fmaf(a[r][i], H[i], x[r][i]);
        A[i] *= a[r][i];
      }
      if (PACKED && p.dfinal && (docs.ends >> r & 1)) {      // the gradient of a final state comes in with the last token
        const int doc = docs.closed(r);
        if (active && doc >= 0)
#pragma unroll
          for (int i = 0; i < VEC; ++i) dh[r][i] += p.dfinal[static_cast<int64_t>(doc) * p.D + c0 + i];
      }
    }
#pragma unroll
    for (int r = SCAN_ROWS - 1; r >= 0; --r)
#pragma unroll
      for (int i = 0; i < VEC; ++i) M[i] = a[r][i] * (PACKED && (docs.ends >> r & 1) ? dh[r][i] : dh[r][i] + M[i]);
    write_map<VEC>(maps.v[buf][0][warp], lane, A);
    write_map<VEC>(maps.v[buf][1][warp], lane, H);
    write_map<VEC>(maps.v[buf][2][warp], lane, M);
    if (PACKED && lane == 0) maps.cut[buf][0][warp] = docs.starts != 0, maps.cut[buf][1][warp] = docs.ends != 0;
    __syncthreads();

    float pa[VEC], ph[VEC], mu[VEC];
    bool cut = false;
#pragma unroll
    for (int i = 0; i < VEC; ++i) pa[i] = 1.f, ph[i] = 0.f;
#pragma unroll
    for (int w = 0; w < SCAN_WARPS; ++w) {
      if (w == warp) break;
      const Channels<VEC> wa = read_map<VEC>(maps.v[buf][0][w], lane), wh = read_map<VEC>(maps.v[buf][1][w], lane);
      const bool wcut = PACKED && maps.cut[buf][0][w];
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        ph[i] = wcut ? wh.v[i] : fmaf(wa.v[i], ph[i], wh.v[i]);
        pa[i] *= wa.v[i];
      }
      cut = cut || wcut;
    }
#pragma unroll
    for (int i = 0; i < VEC; ++i) h[i] = cut ? ph[i] : fmaf(pa[i], h[i], ph[i]);
    cut = false;
#pragma unroll
    for (int i = 0; i < VEC; ++i) pa[i] = 1.f, ph[i] = 0.f, mu[i] = carry[i];
#pragma unroll
    for (int w = SCAN_WARPS - 1; w >= 0; --w) {
      const Channels<VEC> wa = read_map<VEC>(maps.v[buf][0][w], lane), wm = read_map<VEC>(maps.v[buf][2][w], lane);
      const bool wcut = PACKED && maps.cut[buf][1][w];
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        if (w == warp) mu[i] = cut ? ph[i] : fmaf(pa[i], carry[i], ph[i]);
        ph[i] = wcut ? wm.v[i] : fmaf(wa.v[i], ph[i], wm.v[i]);
        pa[i] *= wa.v[i];
      }
      cut = cut || wcut;
    }
#pragma unroll
    for (int i = 0; i < VEC; ++i) carry[i] = cut ? ph[i] : fmaf(pa[i], carry[i], ph[i]);

#pragma unroll
    for (int r = 0; r < SCAN_ROWS; ++r) {        // x becomes the state before its row
      const bool starts = PACKED && (docs.starts >> r & 1);
      float own[VEC];
#pragma unroll
      for (int i = 0; i < VEC; ++i) own[i] = 0.f;
      if (PACKED && starts && p.initial) {
        const int64_t at = static_cast<int64_t>(docs.opened(r)) * p.D + c0;
        if (active)
#pragma unroll
          for (int i = 0; i < VEC; ++i) own[i] = p.initial[at + i];
      }
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        const float before = starts ? own[i] : h[i];
        h[i] = starts ? x[r][i] : fmaf(a[r][i], h[i], x[r][i]);
        x[r][i] = before;
      }
    }
    const int64_t row = (static_cast<int64_t>(b) * p.T + t0) * p.D + c0;
    TX* dx = static_cast<TX*>(p.dx) + row;
    TG* dg = static_cast<TG*>(p.dg) + row;
#pragma unroll
    for (int r = SCAN_ROWS - 1; r >= 0; --r) {
      float lam[VEC], d[VEC];
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        lam[i] = PACKED && (docs.ends >> r & 1) ? dh[r][i] : dh[r][i] + mu[i];
        mu[i] = a[r][i] * lam[i];
        d[i] = mu[i] * x[r][i];
      }
      if (active && t0 + r < p.T) {
        store_pack<TX, VEC>(dx + static_cast<int64_t>(r) * p.D, lam);
        store_pack<TG, VEC>(dg + static_cast<int64_t>(r) * p.D, d);
      }
      if (PACKED && p.dinitial && (docs.starts >> r & 1)) {
        const int doc = docs.opened(r);
        if (active)
#pragma unroll
          for (int i = 0; i < VEC; ++i) p.dinitial[static_cast<int64_t>(doc) * p.D + c0 + i] = mu[i];
      }
    }
  }
  if (!PACKED && p.dinitial && warp == 0 && active)
#pragma unroll
    for (int i = 0; i < VEC; ++i) p.dinitial[static_cast<int64_t>(b) * p.D + c0 + i] = carry[i];
}

// One token: state <- exp(g) state + x in place, h the new state in x's type.  A stream over the state.
template <typename TX, typename TG, int VEC>
__global__ void __launch_bounds__(256)
scan_step_kernel(const TX* x, int64_t x_row, const TG* g, int64_t g_row, float* state, TX* h, int B, int D) {
  const int64_t vectors = static_cast<int64_t>(B) * (D / VEC);
  const int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
  if (i >= vectors) return;
  const int64_t b = i / (D / VEC);
  const int c = static_cast<int>(i - b * (D / VEC)) * VEC;
  const Pack<TX, VEC> xv = load_pack<TX, VEC>(x + b * x_row + c);
  const Pack<TG, VEC> gv = load_pack<TG, VEC>(g + b * g_row + c);
  const Pack<float, VEC> s = load_pack<float, VEC>(state + b * D + c);
  float v[VEC];
#pragma unroll
  for (int k = 0; k < VEC; ++k) v[k] = fmaf(decay(to_f32(gv.v[k])), s.v[k], to_f32(xv.v[k]));
  store_pack<float, VEC>(state + b * D + c, v);
  store_pack<TX, VEC>(h + b * D + c, v);
}

// map[t] = d + 1 where document d opens at token t, else 0; valid = the offsets start at 0, end at T and strictly increase.  Offsets that
// do not are answered by some map of the same form: its T entries hold 0 .. n_docs whatever the offsets are.
__global__ void __launch_bounds__(256)
scan_map_kernel(const void* cu, int is64, int n_docs, int T, int32_t* map, uint8_t* valid) {
  auto at = [&](int i) -> int64_t { return is64 ? static_cast<const int64_t*>(cu)[i] : static_cast<const int32_t*>(cu)[i]; };
  const int t = blockIdx.x * blockDim.x + threadIdx.x;
  if (t < T) {
    int lo = 0, hi = n_docs;                     // the first offset that is not below t is in [lo, hi]
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (at(mid) < t) lo = mid + 1; else hi = mid;
    }
    map[t] = lo < n_docs && at(lo) == t ? lo + 1 : 0;
  }
  if (blockIdx.x == 0) {
    bool good = at(0) == 0 && at(n_docs) == T;
    for (int i = threadIdx.x; i < n_docs; i += blockDim.x) good = good && at(i) < at(i + 1);
    const int all = __syncthreads_and(good);
    if (threadIdx.x == 0) *valid = all ? 1 : 0;
  }
}

}  // namespace tgdn

using namespace tgdn;

namespace {

template <bool BACKWARD, typename TX, typename TG, int VEC, bool PACKED>
int launch_scan(ScanParams p, cudaStream_t s) {
  p.slices = (p.D + 32 * VEC - 1) / (32 * VEC);
  const int64_t blocks = static_cast<int64_t>(p.B) * p.slices;
  if (blocks > 0x7fffffffLL) return TGDN_ERR_SHAPE;
  if constexpr (BACKWARD) scan_bwd_kernel<TX, TG, VEC, PACKED><<<static_cast<unsigned>(blocks), 32 * SCAN_WARPS, 0, s>>>(p);
  else scan_fwd_kernel<TX, TG, VEC, PACKED><<<static_cast<unsigned>(blocks), 32 * SCAN_WARPS, 0, s>>>(p);
  return tgdn_cuda_error(cudaGetLastError());
}

template <bool BACKWARD, typename TX, typename TG>
int launch_scan_of(const ScanParams& p, bool pairs, cudaStream_t s) {
  if (pairs) return p.map ? launch_scan<BACKWARD, TX, TG, 2, true>(p, s) : launch_scan<BACKWARD, TX, TG, 2, false>(p, s);
  return p.map ? launch_scan<BACKWARD, TX, TG, 1, true>(p, s) : launch_scan<BACKWARD, TX, TG, 1, false>(p, s);
}

template <bool BACKWARD>
int launch_scan_any(const ScanParams& p, int xt, int gt, bool pairs, cudaStream_t s) {
  if (xt == TGDN_F32 && gt == TGDN_F32) return launch_scan_of<BACKWARD, float, float>(p, pairs, s);
  if (xt == TGDN_BF16 && gt == TGDN_F32) return launch_scan_of<BACKWARD, __nv_bfloat16, float>(p, pairs, s);
  if (xt == TGDN_BF16 && gt == TGDN_BF16) return launch_scan_of<BACKWARD, __nv_bfloat16, __nv_bfloat16>(p, pairs, s);
  if (xt == TGDN_F16 && gt == TGDN_F32) return launch_scan_of<BACKWARD, __half, float>(p, pairs, s);
  if (xt == TGDN_F16 && gt == TGDN_F16) return launch_scan_of<BACKWARD, __half, __half>(p, pairs, s);
  return TGDN_ERR_TYPE;
}

bool in_pairs(const void* p, int type) { return reinterpret_cast<uintptr_t>(p) % (2 * type_bytes(type)) == 0; }

int scan_checks(const tgdn_rows* x, const tgdn_rows* g, const int32_t* map, int n_docs, int B, int T, int D) {
  if (!x || !g || !x->data || !g->data) return TGDN_ERR_NULL;
  if (B <= 0 || T <= 0 || D <= 0 || (map && (B != 1 || n_docs <= 0))) return TGDN_ERR_SHAPE;
  if (!type_known(x->type) || !type_known(g->type)) return TGDN_ERR_TYPE;
  return 0;
}

}  // namespace

extern "C" int64_t tgdn_scan_carry_floats(int B, int T, int D) {
  return static_cast<int64_t>(B) * ((T + static_cast<int64_t>(SCAN_TILE) - 1) / SCAN_TILE) * D;
}

extern "C" int tgdn_scan_map(const void* cu_seqlens, int cu_is_int64, int n_docs, int T, int32_t* map, uint8_t* valid, void* stream) {
  if (!cu_seqlens || !map || !valid) return TGDN_ERR_NULL;
  if (n_docs <= 0 || T <= 0) return TGDN_ERR_SHAPE;
  if (!tgdn_check_device()) return TGDN_ERR_DEVICE;
  scan_map_kernel<<<T / 256 + (T % 256 != 0), 256, 0, static_cast<cudaStream_t>(stream)>>>(cu_seqlens, cu_is_int64, n_docs, T, map, valid);
  return tgdn_cuda_error(cudaGetLastError());
}

extern "C" int tgdn_scan_fwd(const tgdn_rows* host_x, const tgdn_rows* host_g, const int32_t* map, int n_docs, int B, int T, int D,
                             const float* initial, void* h, float* final_state, float* carry, void* stream) {
  if (const int rc = scan_checks(host_x, host_g, map, n_docs, B, T, D)) return rc;
  if (!h) return TGDN_ERR_NULL;
  if (!tgdn_check_device()) return TGDN_ERR_DEVICE;
  ScanParams p{};
  p.x = {host_x->data, host_x->stride_outer, host_x->stride_inner};
  p.g = {host_g->data, host_g->stride_outer, host_g->stride_inner};
  p.map = map; p.initial = initial; p.h = h; p.final_state = final_state; p.carry = carry;
  p.B = B; p.T = T; p.D = D; p.n_docs = n_docs;
  p.tiles = (T - 1) / SCAN_TILE + 1;
  const bool pairs = D % 2 == 0 && rows_in_vectors(*host_x, 2) && rows_in_vectors(*host_g, 2) && in_pairs(h, host_x->type);
  return launch_scan_any<false>(p, host_x->type, host_g->type, pairs, static_cast<cudaStream_t>(stream));
}

extern "C" int tgdn_scan_bwd(const tgdn_rows* host_x, const tgdn_rows* host_g, const tgdn_rows* host_dh, const int32_t* map, int n_docs,
                             int B, int T, int D, const float* initial, const float* carry, const float* dfinal, void* dx, void* dg,
                             float* dinitial, void* stream) {
  if (const int rc = scan_checks(host_x, host_g, map, n_docs, B, T, D)) return rc;
  if (!host_dh || !host_dh->data || !carry || !dx || !dg) return TGDN_ERR_NULL;
  if (host_dh->type != host_x->type) return TGDN_ERR_TYPE;
  if (!tgdn_check_device()) return TGDN_ERR_DEVICE;
  ScanParams p{};
  p.x = {host_x->data, host_x->stride_outer, host_x->stride_inner};
  p.g = {host_g->data, host_g->stride_outer, host_g->stride_inner};
  p.dh = {host_dh->data, host_dh->stride_outer, host_dh->stride_inner};
  p.map = map; p.initial = initial; p.carry = const_cast<float*>(carry); p.dfinal = dfinal;
  p.dx = dx; p.dg = dg; p.dinitial = dinitial;
  p.B = B; p.T = T; p.D = D; p.n_docs = n_docs;
  p.tiles = (T - 1) / SCAN_TILE + 1;
  const bool pairs = D % 2 == 0 && rows_in_vectors(*host_x, 2) && rows_in_vectors(*host_g, 2) && rows_in_vectors(*host_dh, 2) &&
                     in_pairs(dx, host_x->type) && in_pairs(dg, host_g->type);
  return launch_scan_any<true>(p, host_x->type, host_g->type, pairs, static_cast<cudaStream_t>(stream));
}

namespace {

template <typename TX, typename TG>
int launch_step(const tgdn_rows& x, const tgdn_rows& g, int B, int D, float* state, void* h, cudaStream_t s) {
  const bool fours = D % 4 == 0 && rows_in_vectors(x, 4) && rows_in_vectors(g, 4) && reinterpret_cast<uintptr_t>(state) % 16 == 0 &&
                     reinterpret_cast<uintptr_t>(h) % (4 * sizeof(TX)) == 0;
  const int64_t threads = static_cast<int64_t>(B) * (fours ? D / 4 : D), blocks = (threads + 255) / 256;
  if (blocks > 0x7fffffffLL) return TGDN_ERR_SHAPE;
  const TX* xp = static_cast<const TX*>(x.data);
  const TG* gp = static_cast<const TG*>(g.data);
  if (fours) scan_step_kernel<TX, TG, 4><<<static_cast<unsigned>(blocks), 256, 0, s>>>(xp, x.stride_outer, gp, g.stride_outer, state, static_cast<TX*>(h), B, D);
  else scan_step_kernel<TX, TG, 1><<<static_cast<unsigned>(blocks), 256, 0, s>>>(xp, x.stride_outer, gp, g.stride_outer, state, static_cast<TX*>(h), B, D);
  return tgdn_cuda_error(cudaGetLastError());
}

}  // namespace

extern "C" int tgdn_scan_step(const tgdn_rows* host_x, const tgdn_rows* host_g, int B, int D, float* state, void* h, void* stream) {
  if (const int rc = scan_checks(host_x, host_g, nullptr, 0, B, 1, D)) return rc;
  if (!state || !h) return TGDN_ERR_NULL;
  if (!tgdn_check_device()) return TGDN_ERR_DEVICE;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int xt = host_x->type, gt = host_g->type;
  if (xt == TGDN_F32 && gt == TGDN_F32) return launch_step<float, float>(*host_x, *host_g, B, D, state, h, s);
  if (xt == TGDN_BF16 && gt == TGDN_F32) return launch_step<__nv_bfloat16, float>(*host_x, *host_g, B, D, state, h, s);
  if (xt == TGDN_BF16 && gt == TGDN_BF16) return launch_step<__nv_bfloat16, __nv_bfloat16>(*host_x, *host_g, B, D, state, h, s);
  if (xt == TGDN_F16 && gt == TGDN_F32) return launch_step<__half, float>(*host_x, *host_g, B, D, state, h, s);
  if (xt == TGDN_F16 && gt == TGDN_F16) return launch_step<__half, __half>(*host_x, *host_g, B, D, state, h, s);
  return TGDN_ERR_TYPE;
}
