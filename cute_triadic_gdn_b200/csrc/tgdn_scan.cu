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
#include <type_traits>

#include "tgdn_common.cuh"
#include "tgdn_host.h"
#include "tgdn_kernels.h"
#include "tgdn_rows.cuh"

namespace tgdn {

constexpr int SCAN_ROWS = 16;                    // rows a warp holds
constexpr int SCAN_WARPS = 8;
constexpr int SCAN_MAX_CLUSTER = 8;              // blocks along time that exchange their maps
constexpr int SCAN_TILE = SCAN_ROWS * SCAN_WARPS;
static_assert(SCAN_TILE == TGDN_SCAN_TILE, "rows between two saved states");

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
  void* dx;
  void* dg;
  float* dinitial;
  int B, T, D, n_docs, slices, tiles, cluster, stages;
  int* status;
};

// A lane's channels of one row.  Pairs go through the two-wide f32 instructions: the kernels would be bound by the issue of
// instructions otherwise (one at a time: 37 an element forward, 102 us at 8 x 4096 x 2048 in bf16; see the note at the launch).
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
// to the fifth power is 2^-28 off at 1/8.  (Decays below 2^-126 are zero.)
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
};

// Maps in shared memory, of the block's warps and of the cluster's blocks; double-buffered, so that those of a round are written while
// slower readers are still at the last round's.
template <int VEC, int PARTS, bool PACKED>
struct alignas(16) SharedMaps {
  Lanes<VEC> A[2][PARTS][32], H[2][PARTS][32];
  int cut[2][PARTS];
  __device__ void put(int buf, int part, int lane, const Map<VEC, PACKED>& m) {
    A[buf][part][lane] = m.A;
    H[buf][part][lane] = m.H;
    if (PACKED && lane == 0) cut[buf][part] = m.cut;
  }
  __device__ Map<VEC, PACKED> get(int buf, int part, int lane) const { return {A[buf][part][lane], H[buf][part][lane], PACKED ? cut[buf][part] : 0}; }
};

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t in_block_of_cluster(const void* p, uint32_t rank) {
  uint32_t a;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(p)), "r"(rank));
  return a;
}
// Stores into another block's shared memory that count towards the barrier there with their bytes.
__device__ __forceinline__ void send(uint32_t at, uint32_t bar, uint32_t v) {
  asm volatile("st.async.shared::cluster.mbarrier::complete_tx::bytes.u32 [%0], %1, [%2];" ::"r"(at), "r"(v), "r"(bar) : "memory");
}
__device__ __forceinline__ void send(uint32_t at, uint32_t bar, float v, float w) {
  asm volatile("st.async.shared::cluster.mbarrier::complete_tx::bytes.v2.f32 [%0], {%1, %2}, [%3];" ::"r"(at), "f"(v), "f"(w), "r"(bar) : "memory");
}
__device__ __forceinline__ void send(uint32_t at, uint32_t bar, float a, float b, float c, float d) {
  asm volatile("st.async.shared::cluster.mbarrier::complete_tx::bytes.v4.f32 [%0], {%1, %2, %3, %4}, [%5];"
               ::"r"(at), "f"(a), "f"(b), "f"(c), "f"(d), "r"(bar) : "memory");
}
// The hardware's barrier over the blocks of a cluster, at the kernel's two ends.
__device__ __forceinline__ void cluster_barrier() {
  asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// The maps that the blocks of a cluster send one another, warp k of each to block k.  Two buffers by turns: a block sends its map of round
// n + 2 when it has those of round n + 1, which their blocks sent behind a barrier of all their warps, done with round n.  Messages and a
// barrier on their bytes instead of the cluster's own barrier: that one also waits for the output's stores on their way to memory, 4 us a
// round (packed, 131072 x 1024).
template <int VEC, bool PACKED>
struct ClusterMaps {
  struct alignas(8 * VEC) Entry { Lanes<VEC> A, H; };
  Entry map[2][SCAN_MAX_CLUSTER][32];
  int cut[2][SCAN_MAX_CLUSTER];
  uint64_t full[2];
  static constexpr int BYTES = 32 * sizeof(Entry) + (PACKED ? 4 : 0);          // of one message
  __device__ void init() {
    mbar_init(&full[0], 1);
    mbar_init(&full[1], 1);
    mbar_fence_init();
  }
  // One thread of the block, once a round; messages may come before.
  __device__ void expect(int buf, int blocks) { mbar_expect_tx(&full[buf], blocks * BYTES); }
  __device__ void send_to(int block, int buf, int rank, int lane, const Map<VEC, PACKED>& m) {
    const uint32_t at = in_block_of_cluster(&map[buf][rank][lane], block), bar = in_block_of_cluster(&full[buf], block);
    if constexpr (VEC == 2) send(at, bar, m.A.v[0], m.A.v[1], m.H.v[0], m.H.v[1]);
    else send(at, bar, m.A.v[0], m.H.v[0]);
    if (PACKED && lane == 0) send(in_block_of_cluster(&cut[buf][rank], block), bar, static_cast<uint32_t>(m.cut));
  }
  __device__ void wait(int buf, int turn, const WaitCtl& ctl) { mbar_wait_parked(&full[buf], turn & 1, ctl, DEV_TIMEOUT_LOAD); }
  __device__ Map<VEC, PACKED> get(int buf, int rank, int lane) const {
    const Entry e = map[buf][rank][lane];
    return {e.A, e.H, PACKED ? cut[buf][rank] : 0};
  }
};

// The ring of tiles on their way: stages of shared memory that the copy engine fills, each a block's rows of all its inputs, with a barrier
// that completes when a stage's bytes are in.  One thread asks for a stage again as soon as all warps have what they need of it.
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
};
template <typename TX, typename TG, bool BACKWARD>
struct Ring {
  static constexpr int X_BYTES = SCAN_TILE * 64 * sizeof(TX), G_BYTES = SCAN_TILE * 64 * sizeof(TG);
  static constexpr int BYTES = X_BYTES * (BACKWARD ? 2 : 1) + G_BYTES;
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
      control->abort = 0;
      mbar_fence_init();
    }
    __syncthreads();
  }
  __device__ void request(int t) {
    uint8_t* dst = data + ask * BYTES;
    uint64_t* bar = &control->full[ask];
    mbar_expect_tx(bar, BYTES);
    tma_tile(dst, &maps.x, bar, c, t, b);
    tma_tile(dst + X_BYTES, &maps.g, bar, c, t, b);
    if constexpr (BACKWARD) tma_tile(dst + X_BYTES + G_BYTES, &maps.dh, bar, c, t, b);
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

// Where a block stands: its slice of channels, its batch row, its place in the cluster.
template <int VEC>
struct Place {
  int lane, warp, rank, b, slice0, c0;
  bool active;
  int64_t state;                                 // of the lane's first channel in a (sequences, D) tensor's row b
  __device__ explicit Place(const ScanParams& p) {
    lane = threadIdx.x & 31;
    warp = threadIdx.x >> 5;
    rank = p.cluster > 1 ? static_cast<int>(cluster_rank()) : 0;
    const int unit = blockIdx.x / p.cluster, slice = unit % p.slices;
    b = unit / p.slices;
    slice0 = slice * 32 * VEC;
    c0 = slice0 + lane * VEC;
    active = c0 < p.D;
    state = static_cast<int64_t>(b) * p.D + c0;
  }
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

// RING: pairs of channels, tiles by the copy engine (rows of whole 16-byte pieces).  Otherwise single channels by plain loads of any
// alignment, the next tile in registers.
template <typename TX, typename TG, bool RING, bool PACKED>
__global__ void __launch_bounds__(32 * SCAN_WARPS, sizeof(TX) == 2 ? 2 : 1)
scan_fwd_kernel(const __grid_constant__ ScanMaps tensors, ScanParams p) {
  constexpr int VEC = RING ? 2 : 1;
  using MapT = Map<VEC, PACKED>;
  using BlockMaps = ClusterMaps<VEC, PACKED>;
  extern __shared__ __align__(128) uint8_t dynamic[];
  __shared__ SharedMaps<VEC, SCAN_WARPS, PACKED> maps;
  __shared__ RingControl control;
  BlockMaps& blocks = *reinterpret_cast<BlockMaps*>(dynamic + (RING ? p.stages * Ring<TX, TG, false>::BYTES : 0));
  const Place<VEC> at(p);
  const int lane = at.lane, warp = at.warp, c0 = at.c0;
  const bool active = at.active;
  const int64_t xb = at.b * p.x.sb + (active ? c0 : 0), gb = at.b * p.g.sb + (active ? c0 : 0);
  // the state before the round's tiles, the same in every warp of the cluster
  Lanes<VEC> carry = load_f32<VEC>(p.initial + at.state, !PACKED && p.initial && active);

  const int step = p.cluster * SCAN_TILE, rounds = (p.tiles + p.cluster - 1) / p.cluster, first = at.rank * SCAN_TILE;
  Ring<TX, TG, false> ring(tensors, dynamic, &control, p.status, at.slice0, at.b, RING ? p.stages : 0);
  const bool asks = RING && threadIdx.x == 0;
  if (p.cluster > 1) {
    if (threadIdx.x == 0) blocks.init();
    cluster_barrier();                           // no block sends to another before that one can take it
  }
  RawRows<TX, VEC> xr;
  RawRows<TG, VEC> gr;
  if (asks)
    for (int n = 0; n < p.stages && n < rounds; ++n) ring.request(first + n * step);
  if constexpr (!RING) {
    request_rows<TX>(p.x, xb, first + warp * SCAN_ROWS, p.T, xr);
    request_rows<TG>(p.g, gb, first + warp * SCAN_ROWS, p.T, gr);
  }
  int code = row_code<PACKED>(p, first + warp * SCAN_ROWS, lane);
  for (int round = 0; round < rounds; ++round) {
    const int tile = round * p.cluster + at.rank, t0 = tile * SCAN_TILE + warp * SCAN_ROWS, buf = round & 1;
    Lanes<VEC> a[SCAN_ROWS], x[SCAN_ROWS];
    if (RING) {
      const uint8_t* here = ring.wait();
      take_rows<TX, VEC>(here, warp, lane, xr);
      take_rows<TG, VEC>(here + ring.X_BYTES, warp, lane, gr);
      ring.advance();
    }
    unpack_rows<TX, VEC>(xr, x);
    unpack_rows<TG, VEC>(gr, a);
    if constexpr (!RING)
      if (round + 1 < rounds) {
        request_rows<TX>(p.x, xb, t0 + step, p.T, xr);
        request_rows<TG>(p.g, gb, t0 + step, p.T, gr);
      }
    const RowDocs docs = row_docs<PACKED>(p, t0, code);
    if (round + 1 < rounds) code = row_code<PACKED>(p, t0 + step, lane);
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
    maps.put(buf, warp, lane, run);
    __syncthreads();
    if (asks && round + p.stages < rounds && !ring.given_up()) ring.request(first + (round + p.stages) * step);   // every warp has its rows

    // the maps of the warps before this one, and of all of the block; then the state before the tile
    MapT whole = MapT::identity();
#pragma unroll 2
    for (int w = 0; w < warp; ++w) whole.then(maps.get(buf, w, lane));
    const MapT before = whole;
#pragma unroll 2
    for (int w = warp; w < SCAN_WARPS; ++w) whole.then(maps.get(buf, w, lane));
    Lanes<VEC> mine = carry;
    if (p.cluster > 1) {
      if (warp < p.cluster) blocks.send_to(warp, buf, at.rank, lane, whole);
      if (threadIdx.x == 0) blocks.expect(buf, p.cluster);
      blocks.wait(buf, round >> 1, ring.wait_ctl);
      for (int k = 0; k < p.cluster; ++k) {
        if (k == at.rank) mine = carry;
        blocks.get(buf, k, lane).apply(carry);
      }
    } else {
      whole.apply(carry);
    }
    if (p.carry && warp == 0 && active && tile < p.tiles) store_f32<VEC>(p.carry + (static_cast<int64_t>(at.b) * p.tiles + tile) * p.D + c0, mine);
    before.apply(mine);

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
  if (!PACKED && p.final_state && warp == 0 && at.rank == 0 && active) store_f32<VEC>(p.final_state + at.state, carry);
  if (asks && ring.given_up()) ring.drain();
  if (p.cluster > 1) cluster_barrier();          // a block stays while others may send to it
}

template <typename TX, typename TG, bool RING, bool PACKED>
__global__ void __launch_bounds__(32 * SCAN_WARPS, sizeof(TX) + sizeof(TG) == 4 ? 2 : 1)
scan_bwd_kernel(const __grid_constant__ ScanMaps tensors, ScanParams p) {
  constexpr int VEC = RING ? 2 : 1;
  using MapT = Map<VEC, PACKED>;
  using BlockMaps = ClusterMaps<VEC, PACKED>;
  extern __shared__ __align__(128) uint8_t dynamic[];
  __shared__ SharedMaps<VEC, SCAN_WARPS, PACKED> maps, reverse_maps;
  __shared__ RingControl control;
  BlockMaps& blocks = *reinterpret_cast<BlockMaps*>(dynamic + (RING ? p.stages * Ring<TX, TG, true>::BYTES : 0));
  const Place<VEC> at(p);
  const int lane = at.lane, warp = at.warp, c0 = at.c0;
  const bool active = at.active;
  const int64_t xb = at.b * p.x.sb + (active ? c0 : 0), gb = at.b * p.g.sb + (active ? c0 : 0), hb = at.b * p.dh.sb + (active ? c0 : 0);
  // mu behind the round's tiles, the same in every warp of the cluster
  Lanes<VEC> carry = load_f32<VEC>(p.dfinal + at.state, !PACKED && p.dfinal && active);

  const int step = p.cluster * SCAN_TILE, rounds = (p.tiles + p.cluster - 1) / p.cluster, last = (rounds - 1) * step + at.rank * SCAN_TILE;
  Ring<TX, TG, true> ring(tensors, dynamic, &control, p.status, at.slice0, at.b, RING ? p.stages : 0);
  const bool asks = RING && threadIdx.x == 0;
  if (p.cluster > 1) {
    if (threadIdx.x == 0) blocks.init();
    cluster_barrier();
  }
  RawRows<TX, VEC> xr, hr;
  RawRows<TG, VEC> gr;
  auto request = [&](int t0) {
    if constexpr (!RING) {
      request_rows<TX>(p.x, xb, t0, p.T, xr);
      request_rows<TG>(p.g, gb, t0, p.T, gr);
      request_rows<TX>(p.dh, hb, t0, p.T, hr);
    }
  };
  auto saved = [&](int tile) {                   // the state before a tile
    return load_f32<VEC>(p.carry + (static_cast<int64_t>(at.b) * p.tiles + tile) * p.D + c0, active && tile >= 0 && tile < p.tiles);
  };
  if (asks)
    for (int n = 0; n < p.stages && n < rounds; ++n) ring.request(last - n * step);
  if (!RING) request(last + warp * SCAN_ROWS);
  int code = row_code<PACKED>(p, last + warp * SCAN_ROWS, lane);
  Lanes<VEC> next_h = saved((rounds - 1) * p.cluster + at.rank);
  for (int turn = 0; turn < rounds; ++turn) {
    const int round = rounds - 1 - turn, tile = round * p.cluster + at.rank, t0 = tile * SCAN_TILE + warp * SCAN_ROWS, buf = turn & 1;
    Lanes<VEC> a[SCAN_ROWS], x[SCAN_ROWS], dh[SCAN_ROWS];
    if (RING) {
      const uint8_t* here = ring.wait();
      take_rows<TX, VEC>(here, warp, lane, xr);
      take_rows<TG, VEC>(here + ring.X_BYTES, warp, lane, gr);
      take_rows<TX, VEC>(here + ring.X_BYTES + ring.G_BYTES, warp, lane, hr);
      ring.advance();
    }
    unpack_rows<TX, VEC>(xr, x);
    unpack_rows<TG, VEC>(gr, a);
    unpack_rows<TX, VEC>(hr, dh);
    if (!RING && round > 0) request(t0 - step);
    const RowDocs docs = row_docs<PACKED>(p, t0, code);
    const bool cuts = PACKED && docs.any();
    Lanes<VEC> h = next_h;
    if (round > 0) {
      code = row_code<PACKED>(p, t0 - step, lane);
      next_h = saved(tile - p.cluster);
    }
    decays<VEC>(a);
    MapT run = MapT::identity(), back = run;
    if (cuts) {
      if (p.initial) bring_states<VEC>(p, docs, c0, active, a, x);
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
      run_forward<true, VEC>(docs, a, x, run.A, run.H);
      run_reverse<true, VEC>(docs, a, dh, back.H);
    } else {
      run_forward<false, VEC>(docs, a, x, run.A, run.H);
      run_reverse<false, VEC>(docs, a, dh, back.H);
    }
    back.A = run.A;
    maps.put(buf, warp, lane, run);
    reverse_maps.put(buf, warp, lane, back);
    __syncthreads();
    if (asks && round - p.stages >= 0 && !ring.given_up()) ring.request(last - (turn + p.stages) * step);

    MapT whole = MapT::identity();
#pragma unroll 2
    for (int w = SCAN_WARPS - 1; w > warp; --w) whole.then(reverse_maps.get(buf, w, lane));
    const MapT behind = whole;
#pragma unroll 2
    for (int w = warp; w >= 0; --w) whole.then(reverse_maps.get(buf, w, lane));
    if (p.cluster > 1) {
      if (warp < p.cluster) blocks.send_to(warp, buf, at.rank, lane, whole);
      if (threadIdx.x == 0) blocks.expect(buf, p.cluster);
    }
    MapT before = MapT::identity();
#pragma unroll 2
    for (int w = 0; w < warp; ++w) before.then(maps.get(buf, w, lane));
    before.apply(h);
    if (cuts) {                                  // x becomes the state before its row
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
    if (p.cluster > 1) {
      blocks.wait(buf, turn >> 1, ring.wait_ctl);
      for (int k = p.cluster - 1; k >= 0; --k) {
        if (k == at.rank) mu = carry;
        blocks.get(buf, k, lane).apply(carry);
      }
    } else {
      whole.apply(carry);
    }
    behind.apply(mu);

    const int64_t row = (static_cast<int64_t>(at.b) * p.T + t0) * p.D + c0;
    TX* dx = static_cast<TX*>(p.dx) + row;
    TG* dg = static_cast<TG*>(p.dg) + row;
    const int rows = active ? p.T - t0 : 0, stride = opaque(p.D);
    Lanes<VEC> lam = cuts && docs.ends_at(SCAN_ROWS - 1) ? dh[SCAN_ROWS - 1] : add(dh[SCAN_ROWS - 1], mu);
#pragma unroll
    for (int r = SCAN_ROWS - 1; r >= 0; --r) {
      if (r < SCAN_ROWS - 1) lam = cuts && docs.ends_at(r) ? dh[r] : fma(a[r + 1], lam, dh[r]);
      mu = mul(a[r], lam);
      const Lanes<VEC> d = mul(mu, x[r]);
      if (r < rows) {
        store_f32_as<TX, VEC>(row_of(dx, r, stride), lam.v);
        store_f32_as<TG, VEC>(row_of(dg, r, stride), d.v);
      }
      if (cuts && p.dinitial && docs.starts_at(r)) {
        const int doc = docs.opened(r);
        if (active) store_f32<VEC>(p.dinitial + static_cast<int64_t>(doc) * p.D + c0, mu);
      }
    }
  }
  if (!PACKED && p.dinitial && warp == 0 && at.rank == 0 && active) store_f32<VEC>(p.dinitial + at.state, carry);
  if (asks && ring.given_up()) ring.drain();
  if (p.cluster > 1) cluster_barrier();          // a block stays while others may send to it
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
  Raw<TX, VEC> xr;
  Raw<TG, VEC> gr;
  Raw<float, VEC> sr;
  xr.load(x + b * x_row + c);
  gr.load(g + b * g_row + c);
  sr.load(state + b * D + c);
  float xv[VEC], gv[VEC], v[VEC];
  xr.get(xv);
  gr.get(gv);
  sr.get(v);
#pragma unroll
  for (int k = 0; k < VEC; ++k) v[k] = fmaf(decay<1>(Lanes<1>{{gv[k]}}).v[0], v[k], xv[k]);
  store_f32_as<float, VEC>(state + b * D + c, v);
  store_f32_as<TX, VEC>(h + b * D + c, v);
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

#define TRY_MAP(expr) do { if (const int rc_ = (expr)) return rc_; } while (0)

// A (B, T, D) tensor for the copy engine, tiles of 64 channels of 128 tokens; rows past T and channels past D arrive as zeros.
template <typename T>
int scan_map_of(CUtensorMap* map, const ScanIn& in, int B, int T_, int D) {
  const int64_t row = in.st ? in.st : D;         // an axis of size one has no stride to speak of: any valid one will do
  return tgdn_make_typed_rows_map(map, in.p, sizeof(T) == 4 ? TGDN_F32 : std::is_same<T, __half>::value ? TGDN_F16 : TGDN_BF16, D, T_, B, row,
                                  B > 1 ? in.sb : row * T_, 64, SCAN_TILE);
}

template <bool BACKWARD, typename TX, typename TG, bool RING, bool PACKED>
int launch_scan(ScanParams p, cudaStream_t s) {
  constexpr int VEC = RING ? 2 : 1;
  p.slices = (p.D + 32 * VEC - 1) / (32 * VEC);
  const int64_t units = static_cast<int64_t>(p.B) * p.slices;
  const int sms = tgdn_sm_count();
  p.cluster = 1;
  while (p.cluster < SCAN_MAX_CLUSTER && p.cluster < p.tiles && units * p.cluster * 2 <= sms) p.cluster *= 2;
  if (units * p.cluster > 0x7fffffffLL) return TGDN_ERR_SHAPE;
  constexpr int fixed = (BACKWARD ? 2 : 1) * static_cast<int>(sizeof(SharedMaps<VEC, SCAN_WARPS, PACKED>)) + 256;   // static shared memory, and some
  ScanMaps maps{};
  int bytes = p.cluster > 1 ? static_cast<int>(sizeof(ClusterMaps<VEC, PACKED>)) : 0;
  if constexpr (RING) {
    TRY_MAP(scan_map_of<TX>(&maps.x, p.x, p.B, p.T, p.D));
    TRY_MAP(scan_map_of<TG>(&maps.g, p.g, p.B, p.T, p.D));
    if (BACKWARD) TRY_MAP(scan_map_of<TX>(&maps.dh, p.dh, p.B, p.T, p.D));
    constexpr int stage = Ring<TX, TG, BACKWARD>::BYTES;
    const int two = (228 * 1024 / 2 - 1024 - fixed - bytes) / stage, one = (227 * 1024 - fixed - bytes) / stage;
    // Two blocks an SM wherever two stages leave room: with more blocks than SMs, and in clusters, whose eight blocks must find SMs of one
    // part of the chip free at the same time (packed, 131072 x 1024, 16 clusters: 457 us forward with two stages, 700 with four).
    p.stages = (units * p.cluster > sms || p.cluster > 1) && two >= 2 ? two : one;
    if (p.stages > SCAN_MAX_STAGES) p.stages = SCAN_MAX_STAGES;
    bytes += p.stages * stage;
  }
  auto launch = [&](auto kernel) -> int {
    static bool configured[64] = {false};
    if (const int rc = tgdn_dynamic_smem(reinterpret_cast<const void*>(kernel), 227 * 1024 - fixed, configured)) return rc;
    cudaLaunchConfig_t config{};
    config.gridDim = dim3(static_cast<unsigned>(units * p.cluster));
    config.blockDim = dim3(32 * SCAN_WARPS);
    config.dynamicSmemBytes = bytes;
    config.stream = s;
    cudaLaunchAttribute attribute{};
    attribute.id = cudaLaunchAttributeClusterDimension;
    attribute.val.clusterDim.x = static_cast<unsigned>(p.cluster);
    attribute.val.clusterDim.y = attribute.val.clusterDim.z = 1;
    config.attrs = &attribute;
    config.numAttrs = p.cluster > 1 ? 1 : 0;
    return tgdn_cuda_error(cudaLaunchKernelEx(&config, kernel, maps, p));
  };
  if constexpr (BACKWARD) return launch(scan_bwd_kernel<TX, TG, RING, PACKED>);
  else return launch(scan_fwd_kernel<TX, TG, RING, PACKED>);
}

template <bool BACKWARD, typename TX, typename TG>
int launch_scan_of(const ScanParams& p, bool pieces, cudaStream_t s) {
  if (pieces) return p.map ? launch_scan<BACKWARD, TX, TG, true, true>(p, s) : launch_scan<BACKWARD, TX, TG, true, false>(p, s);
  return p.map ? launch_scan<BACKWARD, TX, TG, false, true>(p, s) : launch_scan<BACKWARD, TX, TG, false, false>(p, s);
}

template <bool BACKWARD>
int launch_scan_any(const ScanParams& p, int xt, int gt, bool pieces, cudaStream_t s) {
  if (xt == TGDN_F32 && gt == TGDN_F32) return launch_scan_of<BACKWARD, float, float>(p, pieces, s);
  if (xt == TGDN_BF16 && gt == TGDN_F32) return launch_scan_of<BACKWARD, __nv_bfloat16, float>(p, pieces, s);
  if (xt == TGDN_BF16 && gt == TGDN_BF16) return launch_scan_of<BACKWARD, __nv_bfloat16, __nv_bfloat16>(p, pieces, s);
  if (xt == TGDN_F16 && gt == TGDN_F32) return launch_scan_of<BACKWARD, __half, float>(p, pieces, s);
  if (xt == TGDN_F16 && gt == TGDN_F16) return launch_scan_of<BACKWARD, __half, __half>(p, pieces, s);
  return TGDN_ERR_TYPE;
}

ScanIn scan_in(const tgdn_rows& t, int T) { return {t.data, t.stride_outer, T == 1 ? 0 : static_cast<int>(t.stride_inner)}; }

// What the copy engine takes: rows of whole 16-byte pieces, axes that advance.  Pairs of the outputs follow from D.
bool in_pieces(const tgdn_rows& t, int B, int T, int D) {
  const int64_t piece = 16 / type_bytes(t.type);
  return reinterpret_cast<uintptr_t>(t.data) % 16 == 0 && D % piece == 0 && (T == 1 || (t.stride_inner > 0 && t.stride_inner % piece == 0)) &&
         (B == 1 || (t.stride_outer > 0 && t.stride_outer % piece == 0 && t.stride_outer < int64_t{1} << 36));
}
bool aligned(const void* p, int bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

int scan_checks(const tgdn_rows* x, const tgdn_rows* g, const int32_t* map, int n_docs, int B, int T, int D) {
  if (!x || !g || !x->data || !g->data) return TGDN_ERR_NULL;
  if (B <= 0 || T <= 0 || T > 0x7fffffff - 2 * SCAN_MAX_CLUSTER * SCAN_TILE || D <= 0 || (map && (B != 1 || n_docs <= 0))) return TGDN_ERR_SHAPE;
  if (!type_known(x->type) || !type_known(g->type)) return TGDN_ERR_TYPE;
  if (x->stride_inner > 0x7fffffffLL || g->stride_inner > 0x7fffffffLL || x->stride_inner < 0 || g->stride_inner < 0) return TGDN_ERR_SHAPE;
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
  p.x = scan_in(*host_x, T);
  p.g = scan_in(*host_g, T);
  p.map = map; p.initial = initial; p.h = h; p.final_state = final_state; p.carry = carry;
  p.B = B; p.T = T; p.D = D; p.n_docs = n_docs;
  p.tiles = (T - 1) / SCAN_TILE + 1;
  const bool pieces = in_pieces(*host_x, B, T, D) && in_pieces(*host_g, B, T, D) && aligned(h, 8);
  p.status = tgdn_status_word();
  return launch_scan_any<false>(p, host_x->type, host_g->type, pieces, static_cast<cudaStream_t>(stream));
}

extern "C" int tgdn_scan_bwd(const tgdn_rows* host_x, const tgdn_rows* host_g, const tgdn_rows* host_dh, const int32_t* map, int n_docs,
                             int B, int T, int D, const float* initial, const float* carry, const float* dfinal, void* dx, void* dg,
                             float* dinitial, void* stream) {
  if (const int rc = scan_checks(host_x, host_g, map, n_docs, B, T, D)) return rc;
  if (!host_dh || !host_dh->data || !carry || !dx || !dg) return TGDN_ERR_NULL;
  if (host_dh->type != host_x->type) return TGDN_ERR_TYPE;
  if (host_dh->stride_inner > 0x7fffffffLL || host_dh->stride_inner < 0) return TGDN_ERR_SHAPE;
  if (!tgdn_check_device()) return TGDN_ERR_DEVICE;
  ScanParams p{};
  p.x = scan_in(*host_x, T);
  p.g = scan_in(*host_g, T);
  p.dh = scan_in(*host_dh, T);
  p.map = map; p.initial = initial; p.carry = const_cast<float*>(carry); p.dfinal = dfinal;
  p.dx = dx; p.dg = dg; p.dinitial = dinitial;
  p.B = B; p.T = T; p.D = D; p.n_docs = n_docs;
  p.tiles = (T - 1) / SCAN_TILE + 1;
  const bool pieces = in_pieces(*host_x, B, T, D) && in_pieces(*host_g, B, T, D) && in_pieces(*host_dh, B, T, D) && aligned(dx, 8) && aligned(dg, 8);
  p.status = tgdn_status_word();
  return launch_scan_any<true>(p, host_x->type, host_g->type, pieces, static_cast<cudaStream_t>(stream));
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
