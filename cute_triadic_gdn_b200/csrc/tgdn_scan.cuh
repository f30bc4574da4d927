// Gated linear recurrence per channel:  h[t] = exp(g[t]) h[t-1] + x[t]  over (B, T, D), forward, backward and one token.
//
// With a = exp(g) a run of rows maps the state c before it to the state behind it by c -> A c + H, A the product of its a and H its own
// result from zero; such maps compose, so the time axis is cut into runs that are walked at the same time.  The gradient runs the other
// way: with lam[t] = dL/dh[t] and mu[t] = a[t] lam[t],
//     lam[t] = dh[t] + mu[t+1],   dx[t] = lam[t],   dg[t] = mu[t] h[t-1],   dinitial = mu[first],
// and a run maps the mu behind it to the mu before it by mu -> A mu + M with the same A.
//
// A warp holds 16 rows of 32 or 64 channels in registers, a block of eight warps a tile of 128 rows.  Two ways over the tiles of a slice of
// channels, with the same arithmetic in the same order:
//   whole    one block walks them with the state in registers: every input is read once, every output written once;
//   split    where slices and batch rows are too few to fill the SMs: the map of every tile (a pass over g and x, or g and dh), the states
//            between the tiles from those (scan_fold_kernel, a walk over two numbers a tile and channel), and the outputs, tiles independent.
// The bound is HBM: 6 bytes an element forward and 10 backward in 16 bits, and two operands more for the split way.  The backward forms h
// again from x and the f32 state before every tile, which the forward leaves (4 bytes per 128 rows and channel): the output in 16 bits would
// put its rounding into dg, and would have to be read in the place of x.
//
// Sums, products and states are f32.  Maps are composed in an order given by the tiles alone, so a sequence's results depend neither on what
// runs beside it nor on the way taken.  Gates above zero may take A out of f32's range where no state leaves it: see "factors out of range".
#pragma once

#include <float.h>
#include <type_traits>

#include "tgdn_common.cuh"
#include "tgdn_host.h"
#include "tgdn_kernels.h"
#include "tgdn_rows.cuh"

namespace tgdn {

constexpr int SCAN_ROWS = 16;                    // rows a warp holds
constexpr int SCAN_WARPS = 8;
constexpr int SCAN_TILE = SCAN_ROWS * SCAN_WARPS;
static_assert(SCAN_TILE == TGDN_SCAN_TILE, "rows between two saved states");

enum ScanWay { SCAN_WHOLE, SCAN_MAPS, SCAN_FINISH };

struct ScanIn {
  const void* p;
  int64_t sb;                                    // elements from one batch row, and from one token, to the next
  int st;
};

struct ScanParams {
  ScanIn x, g, dh;
  const int32_t* map;                            // packed: document + 1 at its first token, 0 elsewhere
  const float* initial;                          // (sequences, D) or nullptr
  const float* dfinal;
  void* h;                                       // forward: output;  backward: unused
  float* final_state;
  float* carry;                                  // (B, tiles, D): the state before every tile
  float* mu;                                     // split backward, the same of mu behind every tile
  float *map_a, *map_h;                          // split: the tiles' maps, (B, tiles, D) each
  int* map_cut;                                  // (tiles): a document's border in the tile
  void* dx;
  void* dg;
  float* dinitial;
  int B, T, D, n_docs, slices, tiles, stages;
  int spans, per_span;                           // a slice's tiles among blocks (whole: one span)
  int* status;
};

// A lane's channels of one row.  Pairs go through the two-wide f32 instructions: with one channel an instruction the forward issues 37 an
// element and is bound by that, with two 21 (8 x 4096 x 2048 in bf16, tiles in registers: 102 and 94 us; by the ring 78).
template <int VEC>
struct alignas(4 * VEC) Lanes {
  float v[VEC];
};
__device__ __forceinline__ float2 pair_of(const Lanes<2>& l) { return make_float2(l.v[0], l.v[1]); }
__device__ __forceinline__ Lanes<2> lanes_of(float2 p) { return {{p.x, p.y}}; }
__device__ __forceinline__ Lanes<2> fma(const Lanes<2>& a, const Lanes<2>& b, const Lanes<2>& c) { return lanes_of(__ffma2_rn(pair_of(a), pair_of(b), pair_of(c))); }
__device__ __forceinline__ Lanes<2> mul(const Lanes<2>& a, const Lanes<2>& b) { return lanes_of(__fmul2_rn(pair_of(a), pair_of(b))); }
__device__ __forceinline__ Lanes<2> add(const Lanes<2>& a, const Lanes<2>& b) { return lanes_of(__fadd2_rn(pair_of(a), pair_of(b))); }
__device__ __forceinline__ Lanes<1> fma(const Lanes<1>& a, const Lanes<1>& b, const Lanes<1>& c) { return {{fmaf(a.v[0], b.v[0], c.v[0])}}; }
__device__ __forceinline__ Lanes<1> mul(const Lanes<1>& a, const Lanes<1>& b) { return {{__fmul_rn(a.v[0], b.v[0])}}; }
__device__ __forceinline__ Lanes<1> add(const Lanes<1>& a, const Lanes<1>& b) { return {{__fadd_rn(a.v[0], b.v[0])}}; }
template <int VEC>
__device__ __forceinline__ Lanes<VEC> all(float f) {
  Lanes<VEC> r;
#pragma unroll
  for (int i = 0; i < VEC; ++i) r.v[i] = f;
  return r;
}
template <int VEC>
__device__ __forceinline__ Lanes<VEC> load_f32(const float* p, bool ok) {
  Lanes<VEC> r;
#pragma unroll
  for (int i = 0; i < VEC; ++i) r.v[i] = ok ? p[i] : 0.f;
  return r;
}
template <int VEC>
__device__ __forceinline__ void store_f32(float* p, const Lanes<VEC>& l) {
#pragma unroll
  for (int i = 0; i < VEC; ++i) p[i] = l.v[i];
}

__device__ __forceinline__ float power_of_two(float t) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(t));
  return r;
}
// exp(g).  Near zero as 1 + (g + g^2/2 + ...): the sum is rounded once, to nearest, while the hardware's power of two errs by up to two
// units to one side, and such errors add up over as many tokens as the state remembers (a thousand tokens at g = -1e-3: 2e-5 where
// roundings to nearest leave 1e-6).  Beyond 1/8 a state remembers eight tokens at most and the power of two is good enough.  The series
// to the fifth power is 2^-27.3 off at -1/8, a tenth of a rounding's 2^-24, and 2^-33.4 at -1/16.  (Decays below 2^-126 are zero.)
template <int VEC>
__device__ __forceinline__ Lanes<VEC> decay(const Lanes<VEC>& g) {
  Lanes<VEC> s = fma(g, all<VEC>(1.f / 120.f), all<VEC>(1.f / 24.f));
  s = fma(g, s, all<VEC>(1.f / 6.f));
  s = fma(g, s, all<VEC>(0.5f));
  s = fma(g, s, all<VEC>(1.f));
  s = fma(g, s, all<VEC>(1.f));
  const Lanes<VEC> t = mul(g, all<VEC>(1.4426950408889634f));
#pragma unroll
  for (int i = 0; i < VEC; ++i) s.v[i] = fabsf(g.v[i]) < 0.125f ? s.v[i] : power_of_two(t.v[i]);
  return s;
}
// The same for the rows of a tile; single channels two rows at a time.
template <int VEC>
__device__ __forceinline__ void decays(Lanes<VEC> (&g)[SCAN_ROWS]) {
  if constexpr (VEC == 1) {
#pragma unroll
    for (int r = 0; r < SCAN_ROWS; r += 2) {
      const Lanes<2> a = decay<2>(Lanes<2>{{g[r].v[0], g[r + 1].v[0]}});
      g[r].v[0] = a.v[0], g[r + 1].v[0] = a.v[1];
    }
  } else {
#pragma unroll
    for (int r = 0; r < SCAN_ROWS; ++r) g[r] = decay<VEC>(g[r]);
  }
}

// What a warp knows about the documents of its rows: bit r of `starts`, row r opens a document (whose number + 1 lane r holds); bit r of
// `ends`, it closes one.
struct RowDocs {
  uint32_t starts, ends;
  int code;
  __device__ bool any() const { return (starts | ends) != 0; }
  __device__ bool starts_at(int r) const { return starts >> r & 1; }
  __device__ bool ends_at(int r) const { return ends >> r & 1; }
  __device__ int opened(int r) const { return __shfl_sync(0xffffffffu, code, r) - 1; }
  // The document before the one that opens at the next row; -1 where offsets that do not start at 0 leave none.
  __device__ int closed(int r) const { return __shfl_sync(0xffffffffu, code, r + 1) - 2; }
};

// The lane's entry of the map for the rows from t0 on (and the one behind them): asked for a round ahead.
template <bool PACKED>
__device__ __forceinline__ int row_code(const ScanParams& p, int t0, int lane) {
  const int t = t0 + lane;
  return !PACKED || lane > SCAN_ROWS || t > p.T ? 0 : t == p.T ? p.n_docs + 1 : p.map[t];
}
template <bool PACKED>
__device__ __forceinline__ RowDocs row_docs(const ScanParams& p, int t0, int code) {
  RowDocs d{0u, 0u, code};
  if constexpr (PACKED) {
    const uint32_t b = __ballot_sync(0xffffffffu, code != 0);
    d.starts = b & ((1u << SCAN_ROWS) - 1);
    if (t0 + SCAN_ROWS > p.T && t0 <= p.T) d.starts &= (1u << (p.T - t0)) - 1;
    d.ends = (b >> 1) & ((1u << SCAN_ROWS) - 1);
  }
  return d;
}

// A tile's rows as they lie in memory: what a warp has in flight while it works on the tile before.
template <typename T, int VEC>
struct RawRows {
  Raw<T, VEC> v[SCAN_ROWS];
};

// Reads that nothing else in the kernel writes, in the order they stand in (volatile: they must be under way before the work that hides
// them), and past L1: no line is read twice by a block.
template <typename T>
__device__ __forceinline__ void read_once(Raw<T, 1>& d, const T* p) {
  if constexpr (sizeof(T) == 4) {
    asm volatile("ld.global.nc.L1::no_allocate.b32 %0, [%1];" : "=r"(d.w[0]) : "l"(p));
  } else {
    uint16_t v;
    asm volatile("ld.global.nc.L1::no_allocate.b16 %0, [%1];" : "=h"(v) : "l"(p));
    d.w[0] = v;
  }
}

// Row r of a tile, for a stride below 2^31 elements (the launch checks): one wide product an address.  `stride` is made opaque once a tile, or
// the compiler would keep its sixteen multiples in registers across the loop.
template <typename T>
__device__ __forceinline__ T* row_of(T* p, int r, int stride) { return p + static_cast<int64_t>(r) * stride; }
__device__ __forceinline__ int opaque(int v) {
  asm volatile("" : "+r"(v));
  return v;
}

// Rows past T read as zeros.  Lanes past D read channel 0 (`base` says so) and store nothing.
template <typename T>
__device__ __forceinline__ void request_rows(const ScanIn& in, int64_t base, int t0, int T_, RawRows<T, 1>& raw) {
  const T* p = static_cast<const T*>(in.p) + base + static_cast<int64_t>(t0) * in.st;
  const int rows = T_ - t0, stride = opaque(in.st);
  if (rows >= SCAN_ROWS) {
#pragma unroll
    for (int r = 0; r < SCAN_ROWS; ++r) read_once(raw.v[r], row_of(p, r, stride));
  } else {
#pragma unroll
    for (int r = 0; r < SCAN_ROWS; ++r) {
      raw.v[r].zero();
      if (r < rows) read_once(raw.v[r], row_of(p, r, stride));
    }
  }
}
template <typename T, int VEC>
__device__ __forceinline__ void unpack_rows(const RawRows<T, VEC>& raw, Lanes<VEC> (&out)[SCAN_ROWS]) {
#pragma unroll
  for (int r = 0; r < SCAN_ROWS; ++r) raw.v[r].get(out[r].v);
}

// Factors out of range.  With gates above zero the product A of a run's decays may pass 2^128 where the states stay small, or zero, or shrink
// again within the run.  A factor is never negative, so that one from 2^128 up to 2^319 is written as -A 2^-192; beyond that the smallest
// state but zero overflows, and A is +infinity.  The blocks compose plainly, note in shared memory where a run's factor passes 2^15 (eight of
// up to 2^15 stay in range in whatever order they are composed) and then walk their tiles once more by the wide forms: the same arithmetic
// on plain factors, in the same order, 64 bits on the others.  (A test within the walk, with a branch, cost blocks that are alone on their
// SM a third: 1 x 4096 x 4096 in bf16, backward, 72 -> 98 us; the note costs 0 to 2 %.  Where all
// blocks walk twice, 8 x 4096 x 2048 takes 181 / 308 us instead of 76 / 136.)  Limits that remain: exp(g) is f32, and what is below
// 2^-126, a state or a product of decays, counts as zero.
__device__ __forceinline__ bool plain_factor(float a) { return a >= 0.f && a <= FLT_MAX; }
__device__ __forceinline__ double factor_value(float a) { return a < 0.f ? static_cast<double>(a) * -0x1p192 : static_cast<double>(a); }
__device__ __forceinline__ float factor_of(double v) {
  if (!(v > FLT_MAX)) return static_cast<float>(v);
  const float scaled = static_cast<float>(v * 0x1p-192);
  return scaled <= FLT_MAX ? -scaled : scaled;
}
__device__ __forceinline__ float factor_times(float a, float b) {
  const float product = a * b;
  if (plain_factor(a) && plain_factor(b) && product <= FLT_MAX) return product;
  if (a == 0.f) return b == b ? 0.f : b;         // (no 0 x infinity: what has come to zero does not grow, and what overflows stays so)
  if (isinf(a)) return b == b ? a : b;
  return factor_of(factor_value(a) * factor_value(b));
}
__device__ __forceinline__ float factor_apply(float a, float c, float h) {
  if (plain_factor(a) || a != a) return fmaf(a, c, h);
  if (c == 0.f) return h;
  return isinf(a) ? fmaf(a, c, h) : static_cast<float>(factor_value(a) * c + h);
}
// The product of a run's decays where the plain one left the range on its way: exponents by steps of 2^64 beside the number.
template <int VEC>
__device__ __forceinline__ float factor_of_run(const Lanes<VEC> (&a)[SCAN_ROWS], int i) {
  float m = 1.f;
  int e = 0;
#pragma unroll
  for (int r = 0; r < SCAN_ROWS; ++r) {
    const bool steep = a[r].v[i] > 0x1p32f, high = m > 0x1p32f, low = m < 0x1p-32f && e > 0;
    m = (high ? m * 0x1p-64f : low ? m * 0x1p64f : m) * (steep ? a[r].v[i] * 0x1p-64f : a[r].v[i]);
    e += steep + high - low;
  }
  double v = m;
  for (; e > 0 && v <= 0x1p400; --e) v *= 0x1p64;
  return factor_of(v);
}

// A map of a run of rows in a lane's channels: c -> A c + H, or c -> H where a document's border lies in the run (`cut`, one value for all
// channels: a state that is infinite or NaN must not pass, so a factor of zero would not do).
template <int VEC, bool PACKED>
struct Map {
  Lanes<VEC> A, H;
  int cut;
  __device__ static Map identity() { return Map{all<VEC>(1.f), all<VEC>(0.f), 0}; }
  __device__ void then(const Map& n) {           // this map, then n
    H = PACKED && n.cut ? n.H : fma(n.A, H, n.H);
    A = mul(A, n.A);
    if (PACKED) cut |= n.cut;
  }
  __device__ void apply(Lanes<VEC>& c) const { c = PACKED && cut ? H : fma(A, c, H); }
  __device__ bool moderate() const {             // (false for NaN)
    bool all = A.v[0] <= 0x1p15f;
#pragma unroll
    for (int i = 1; i < VEC; ++i) all = all && A.v[i] <= 0x1p15f;
    return all;
  }
  // The same with factors of any size: the run's own product `of` its decays, this map, then n, and a state through the map.
  __device__ void widen(const Lanes<VEC> (&of)[SCAN_ROWS]) {
#pragma unroll
    for (int i = 0; i < VEC; ++i)
      if (!plain_factor(A.v[i])) A.v[i] = factor_of_run<VEC>(of, i);
  }
  __device__ void then_wide(const Map& n) {
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      H.v[i] = PACKED && n.cut ? n.H.v[i] : factor_apply(n.A.v[i], H.v[i], n.H.v[i]);
      A.v[i] = factor_times(A.v[i], n.A.v[i]);
    }
    if (PACKED) cut |= n.cut;
  }
  __device__ void apply_wide(Lanes<VEC>& c) const {
#pragma unroll
    for (int i = 0; i < VEC; ++i) c.v[i] = PACKED && cut ? H.v[i] : factor_apply(A.v[i], c.v[i], H.v[i]);
  }
};

// Maps in shared memory, of the block's warps; double-buffered, so that those of a tile are written while slower readers are still at the
// last one's.
template <int VEC, bool PACKED>
struct alignas(16) SharedMaps {
  Lanes<VEC> A[2][SCAN_WARPS][32], H[2][SCAN_WARPS][32];
  int cut[2][SCAN_WARPS];
  __device__ void put(int buf, int part, int lane, const Map<VEC, PACKED>& m) {
    A[buf][part][lane] = m.A;
    H[buf][part][lane] = m.H;
    if (PACKED && lane == 0) cut[buf][part] = m.cut;
  }
  // CUTS: a document's border lies in the tile.
  template <bool CUTS>
  __device__ Map<VEC, CUTS> get(int buf, int part, int lane) const { return {A[buf][part][lane], H[buf][part][lane], CUTS ? cut[buf][part] : 0}; }
};
// The block's barrier between the maps' being written and read; true where a run of the tile holds a document's border.  The tiles that hold none do
// without the selections and their registers (one packed row of 16384 x 8192 in bf16, forward: 313 -> 238 us; 8192 x 16384: 234 -> 176 us).
template <bool PACKED>
__device__ __forceinline__ bool maps_written(bool cut) {
  if constexpr (PACKED) return __syncthreads_or(cut) != 0;
  __syncthreads();
  return false;
}
// f(true) for a tile with a document's border in it, else f(false), as constants.
template <bool PACKED, typename F>
__device__ __forceinline__ void by_cuts(bool cuts, F f) {
  if constexpr (PACKED) {
    if (cuts) {
      f(std::true_type{});
      return;
    }
  }
  f(std::false_type{});
}

// The ring of tiles on their way: two to four stages of shared memory that the copy engine fills, each a block's rows of all its inputs, with
// a barrier that completes when a stage's bytes are in.  One thread asks for a stage again as soon as all warps have what they need of it.
// 64 to 196 KB of an SM's memory are under way so, where a tile in registers was 32 (8 x 4096 x 2048 in bf16: 94 -> 78 us forward, 174 -> 139
// backward, of which 63 and 104 are the bytes at the copy rate; 4 x 4096 x 4096 with f32 gates: 129 -> 92 of 84).
constexpr int SCAN_MAX_STAGES = 4;
__device__ __forceinline__ void tma_tile(void* dst, const CUtensorMap* map, uint64_t* bar, int c, int t, int b) {
  asm volatile("cp.async.bulk.tensor.3d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
               ::"r"(smem_u32(dst)), "l"(map), "r"(smem_u32(bar)), "r"(c), "r"(t), "r"(b)
               : "memory");
}
struct ScanMaps {
  CUtensorMap x, g, dh;
};
struct RingControl {
  uint64_t full[SCAN_MAX_STAGES];
  int abort;
  int wide;                                      // a run's factor was too large for the plain forms
};
template <typename TX, typename TG, bool HAS_X, bool HAS_DH>
struct Ring {
  static constexpr int X_BYTES = SCAN_TILE * 64 * sizeof(TX), G_BYTES = SCAN_TILE * 64 * sizeof(TG);
  static constexpr int X_AT = G_BYTES, DH_AT = G_BYTES + (HAS_X ? X_BYTES : 0), BYTES = DH_AT + (HAS_DH ? X_BYTES : 0);   // g first
  const ScanMaps& maps;
  uint8_t* data;
  RingControl* control;
  WaitCtl wait_ctl;
  int c, b, stages;
  int stage = 0, parity = 0;                     // of the tile that is read next
  int ask = 0, asked = 0;                        // the stage that is asked for next, and how many were (the asking thread's)

  __device__ Ring(const ScanMaps& m, uint8_t* smem, RingControl* ctl, int* status, int c_, int b_, int stages_)
      : maps(m), data(smem), control(ctl), wait_ctl{&ctl->abort, status}, c(c_), b(b_), stages(stages_) {
    if (threadIdx.x == 0) {
      for (int i = 0; i < stages; ++i) mbar_init(&control->full[i], 1);
      control->abort = control->wide = 0;
      mbar_fence_init();
    }
    __syncthreads();
  }
  __device__ void request(int t) {
    uint8_t* dst = data + ask * BYTES;
    uint64_t* bar = &control->full[ask];
    mbar_expect_tx(bar, BYTES);
    tma_tile(dst, &maps.g, bar, c, t, b);
    if constexpr (HAS_X) tma_tile(dst + X_AT, &maps.x, bar, c, t, b);
    if constexpr (HAS_DH) tma_tile(dst + DH_AT, &maps.dh, bar, c, t, b);
    ask = ask + 1 == stages ? 0 : ask + 1;
    ++asked;
  }
  __device__ const uint8_t* wait() const {
    mbar_wait_parked(&control->full[stage], parity, wait_ctl, DEV_TIMEOUT_LOAD);
    return data + stage * BYTES;
  }
  __device__ void advance() {
    if (++stage == stages) stage = 0, parity ^= 1;
  }
  // After a wait that was given up: nothing more is asked for, and what was must have landed before the block's memory goes.
  __device__ bool given_up() const { return *wait_ctl.abort != 0; }
  __device__ void drain() const {
    int none = 0;
    const WaitCtl again{&none, wait_ctl.status};
    for (int n = asked > stages ? asked - stages : 0; n < asked; ++n) mbar_wait_parked(&control->full[n % stages], n / stages & 1, again, DEV_TIMEOUT_LOAD);
  }
};
// A warp's rows of a tile in the ring, as they lie there.
template <typename T, int VEC>
__device__ __forceinline__ void take_rows(const uint8_t* tile, int warp, int lane, RawRows<T, VEC>& raw) {
  const T* p = reinterpret_cast<const T*>(tile) + (warp * SCAN_ROWS * 32 + lane) * VEC;
#pragma unroll
  for (int r = 0; r < SCAN_ROWS; ++r) raw.v[r].load(p + r * 32 * VEC);
}

// Where a block stands: its slice of channels, its batch row, its tiles.
template <int VEC>
struct Place {
  int lane, warp, b, slice0, c0, lo, hi;
  bool active;
  int64_t state;                                 // of the lane's first channel in a (sequences, D) tensor's row b
  // `last_first`: the second pass over the data begins where the first one ended, with what L2 still holds.
  __device__ Place(const ScanParams& p, bool last_first) {
    lane = threadIdx.x & 31;
    warp = threadIdx.x >> 5;
    const int block = last_first ? gridDim.x - 1 - blockIdx.x : blockIdx.x, unit = block / p.spans, slice = unit % p.slices;
    lo = (block - unit * p.spans) * p.per_span;
    hi = min(lo + p.per_span, p.tiles);
    b = unit / p.slices;
    slice0 = slice * 32 * VEC;
    c0 = slice0 + lane * VEC;
    active = c0 < p.D;
    state = static_cast<int64_t>(b) * p.D + c0;
  }
  // Of the lane's first channel in a (B, tiles, D) tensor.
  __device__ int64_t at_tile(const ScanParams& p, int tile) const { return (static_cast<int64_t>(b) * p.tiles + tile) * p.D + c0; }
};

// A run's map from zero, its rows already with the states that documents bring.  CUTS: a document opens or closes in the run; the warps
// that hold none (documents are longer than sixteen tokens as a rule) do without the selections.
template <bool CUTS, int VEC>
__device__ __forceinline__ void run_forward(const RowDocs& docs, const Lanes<VEC> (&a)[SCAN_ROWS], const Lanes<VEC> (&x)[SCAN_ROWS], Lanes<VEC>& A,
                                            Lanes<VEC>& H) {
#pragma unroll
  for (int r = 0; r < SCAN_ROWS; ++r) {
    H = CUTS && docs.starts_at(r) ? x[r] : fma(a[r], H, x[r]);
    A = mul(A, a[r]);
  }
}
// lam of row r from the one behind it; where a document ends in the row nothing comes from behind.
template <bool CUTS, int VEC>
__device__ __forceinline__ void run_reverse(const RowDocs& docs, const Lanes<VEC> (&a)[SCAN_ROWS], const Lanes<VEC> (&dh)[SCAN_ROWS], Lanes<VEC>& M) {
  Lanes<VEC> lam = dh[SCAN_ROWS - 1];
#pragma unroll
  for (int r = SCAN_ROWS - 2; r >= 0; --r) lam = CUTS && docs.ends_at(r) ? dh[r] : fma(a[r + 1], lam, dh[r]);
  M = mul(a[0], lam);
}
// The documents that open in a run bring their own states in with their first tokens.
template <int VEC>
__device__ __forceinline__ void bring_states(const ScanParams& p, const RowDocs& docs, int c0, bool active, const Lanes<VEC> (&a)[SCAN_ROWS],
                                             Lanes<VEC> (&x)[SCAN_ROWS]) {
#pragma unroll
  for (int r = 0; r < SCAN_ROWS; ++r)
    if (docs.starts_at(r)) x[r] = fma(a[r], load_f32<VEC>(p.initial + static_cast<int64_t>(docs.opened(r)) * p.D + c0, active), x[r]);
}

// The maps of the warps from one to before another (BACK: from one back to behind another), composed in order.
template <bool BACK, bool CUTS, int VEC, bool PACKED>
__device__ __forceinline__ void compose(Map<VEC, CUTS>& m, const SharedMaps<VEC, PACKED>& maps, int buf, int lane, int from, int to) {
  if (BACK) {
#pragma unroll 2
    for (int w = from; w > to; --w) m.then(maps.template get<CUTS>(buf, w, lane));
  } else {
#pragma unroll 2
    for (int w = from; w < to; ++w) m.then(maps.template get<CUTS>(buf, w, lane));
  }
}
// The same with the maps of all warps in registers first, which does not wait for shared memory at every step: where registers allow it (the
// forward without a document's border: single channels 10 % faster, pairs 3 %; the backward would spill, 68 -> 90 us at 64 channels x 4096).
template <int VEC, bool CUTS>
struct AllMaps {
  Map<VEC, CUTS> m[SCAN_WARPS];
  template <bool PACKED>
  __device__ AllMaps(const SharedMaps<VEC, PACKED>& maps, int buf, int lane) {
#pragma unroll
    for (int w = 0; w < SCAN_WARPS; ++w) m[w] = maps.template get<CUTS>(buf, w, lane);
  }
  __device__ void compose(Map<VEC, CUTS>& to, int lo, int hi) const {
#pragma unroll
    for (int w = 0; w < SCAN_WARPS; ++w)
      if (w >= lo && w < hi) to.then(m[w]);
  }
};
// The same on factors of any size: the map of the warps [from, to), and the state `at_warp` behind those before `warp` from the state c before all.
template <bool BACK, int VEC, bool CUTS, bool PACKED>
__device__ __forceinline__ Map<VEC, CUTS> compose_wide(const SharedMaps<VEC, PACKED>& maps, int buf, int lane, int from, int to, int warp, const Lanes<VEC>& c,
                                                       Lanes<VEC>& at_warp) {
  Map<VEC, CUTS> m = Map<VEC, CUTS>::identity();
#pragma unroll 1
  for (int w = from;; w += BACK ? -1 : 1) {
    if (w == warp) {
      at_warp = c;
      m.apply_wide(at_warp);
    }
    if (w == to) return m;
    m.then_wide(maps.template get<CUTS>(buf, w, lane));
  }
}
template <int VEC, bool CUTS>
__device__ __forceinline__ void leave_map(const ScanParams& p, const Place<VEC>& at, int tile, const Map<VEC, CUTS>& m) {
  if (at.active) {
    store_f32<VEC>(p.map_a + at.at_tile(p, tile), m.A);
    store_f32<VEC>(p.map_h + at.at_tile(p, tile), m.H);
  }
  if (p.map_cut && at.slice0 == 0 && at.lane == 0) p.map_cut[tile] = CUTS ? m.cut : 0;
}

}  // namespace tgdn

// The launches, by file: the way over the tiles, pieces of 16 bytes (the copy engine) or any alignment.
int tgdn_scan_launch_fwd(const tgdn::ScanParams& p, int x_type, int g_type, bool pieces, tgdn::ScanWay way, cudaStream_t s);
int tgdn_scan_launch_bwd(const tgdn::ScanParams& p, int x_type, int g_type, bool pieces, tgdn::ScanWay way, cudaStream_t s);

namespace tgdn {
namespace {

// A (B, T, D) tensor for the copy engine, tiles of 64 channels of 128 tokens; rows past T and channels past D arrive as zeros.
template <typename T>
int scan_map_of(CUtensorMap* map, const ScanIn& in, int B, int T_, int D) {
  const int64_t row = in.st ? in.st : D;         // an axis of size one has no stride to speak of: any valid one will do
  return tgdn_make_typed_rows_map(map, in.p, sizeof(T) == 4 ? TGDN_F32 : std::is_same<T, __half>::value ? TGDN_F16 : TGDN_BF16, D, T_, B, row,
                                  B > 1 ? in.sb : row * T_, 64, SCAN_TILE);
}

// `fixed`: static shared memory.  Two blocks an SM where the kernel has the registers for it (PER_SM), there are more blocks than SMs and two stages
// leave room.
template <bool RING, typename TX, typename TG, bool HAS_X, bool HAS_DH, int PER_SM, typename Kernel>
int scan_launch(Kernel kernel, bool* configured, int fixed, ScanParams p, cudaStream_t s) {
  ScanMaps maps{};
  int bytes = 0;
  const int64_t blocks = static_cast<int64_t>(p.B) * p.slices * p.spans;
  if (blocks > 0x7fffffffLL) return TGDN_ERR_SHAPE;
  if constexpr (RING) {
    if (const int rc = scan_map_of<TG>(&maps.g, p.g, p.B, p.T, p.D)) return rc;
    if (HAS_X)
      if (const int rc = scan_map_of<TX>(&maps.x, p.x, p.B, p.T, p.D)) return rc;
    if (HAS_DH)
      if (const int rc = scan_map_of<TX>(&maps.dh, p.dh, p.B, p.T, p.D)) return rc;
    constexpr int stage = Ring<TX, TG, HAS_X, HAS_DH>::BYTES;
    const int two = (228 * 1024 / 2 - 1024 - fixed) / stage, one = (227 * 1024 - fixed) / stage;
    p.stages = PER_SM == 2 && blocks > tgdn_sm_count() && two >= 2 ? two : one;
    if (p.stages > SCAN_MAX_STAGES) p.stages = SCAN_MAX_STAGES;
    bytes = p.stages * stage;
    if (const int rc = tgdn_dynamic_smem(reinterpret_cast<const void*>(kernel), 227 * 1024 - fixed, configured)) return rc;
  }
  kernel<<<static_cast<unsigned>(blocks), 32 * SCAN_WARPS, bytes, s>>>(maps, p);
  return tgdn_cuda_error(cudaGetLastError());
}

// The kernels by type, alignment and rows (Launch::go<TX, TG, RING, PACKED>).
template <typename Launch, typename TX, typename TG>
int scan_launch_of(const ScanParams& p, bool pieces, cudaStream_t s) {
  if (pieces) return p.map ? Launch::template go<TX, TG, true, true>(p, s) : Launch::template go<TX, TG, true, false>(p, s);
  return p.map ? Launch::template go<TX, TG, false, true>(p, s) : Launch::template go<TX, TG, false, false>(p, s);
}
template <typename Launch>
int scan_launch_any(const ScanParams& p, int xt, int gt, bool pieces, cudaStream_t s) {
  if (xt == TGDN_F32 && gt == TGDN_F32) return scan_launch_of<Launch, float, float>(p, pieces, s);
  if (xt == TGDN_BF16 && gt == TGDN_F32) return scan_launch_of<Launch, __nv_bfloat16, float>(p, pieces, s);
  if (xt == TGDN_BF16 && gt == TGDN_BF16) return scan_launch_of<Launch, __nv_bfloat16, __nv_bfloat16>(p, pieces, s);
  if (xt == TGDN_F16 && gt == TGDN_F32) return scan_launch_of<Launch, __half, float>(p, pieces, s);
  if (xt == TGDN_F16 && gt == TGDN_F16) return scan_launch_of<Launch, __half, __half>(p, pieces, s);
  return TGDN_ERR_TYPE;
}

}  // namespace
}  // namespace tgdn
