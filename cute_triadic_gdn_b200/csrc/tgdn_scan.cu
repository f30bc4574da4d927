// The gated scan's entry points (tgdn_scan.cuh), the states between the tiles on the split way, one token on a resident state, and the map
// of a packed row's documents.
#include "tgdn_scan.cuh"

namespace tgdn {

// The states between the tiles from the tiles' maps: carry[i] = the state before tile i (REVERSE: behind it), end = the state behind the last
// (before the first).  A block has 32 channels of a batch row; all warps bring the maps of 64 tiles at a time into shared memory, three
// lots ahead, and the first walks over them: a fused multiply-add a tile, 1024 tiles of 1024 channels in 26 us with cold
// caches (a thirtieth of the forward and backward around it; 24 without the look at the factors' range).
constexpr int FOLD_TILES = 64, FOLD_STAGES = 4, FOLD_THREADS = 256;
struct FoldStage {
  float A[FOLD_TILES][32], H[FOLD_TILES][32];
  int cut[FOLD_TILES];
};
__device__ __forceinline__ void copy_word(void* dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
}
template <bool REVERSE>
__global__ void __launch_bounds__(FOLD_THREADS)
scan_fold_kernel(const float* A, const float* H, const int* cut, const float* start, float* carry, float* end, int tiles, int D) {
  extern __shared__ __align__(16) uint8_t dynamic[];
  FoldStage* stages = reinterpret_cast<FoldStage*>(dynamic);
  const int slices = (D + 31) / 32, b = blockIdx.x / slices, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int c = (blockIdx.x - b * slices) * 32 + lane, lots = (tiles + FOLD_TILES - 1) / FOLD_TILES;
  const bool active = c < D;
  const int64_t base = static_cast<int64_t>(b) * tiles * D + c;
  auto tile_of = [&](int i) { return REVERSE ? tiles - 1 - i : i; };
  auto request = [&](int lot) {
    if (lot < lots) {
      FoldStage& s = stages[lot % FOLD_STAGES];
      for (int i = warp; i < FOLD_TILES; i += FOLD_THREADS / 32) {
        const int n = lot * FOLD_TILES + i;
        if (n < tiles && active) {
          copy_word(&s.A[i][lane], A + base + static_cast<int64_t>(tile_of(n)) * D);
          copy_word(&s.H[i][lane], H + base + static_cast<int64_t>(tile_of(n)) * D);
        }
      }
      if (cut)
        for (int i = threadIdx.x; i < FOLD_TILES; i += FOLD_THREADS)
          if (lot * FOLD_TILES + i < tiles) copy_word(&s.cut[i], cut + tile_of(lot * FOLD_TILES + i));
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  for (int lot = 0; lot < FOLD_STAGES - 1; ++lot) request(lot);
  float* out = carry + base + static_cast<int64_t>(tile_of(0)) * D;
  const int64_t step = REVERSE ? -static_cast<int64_t>(D) : D;
  float state = start && active ? start[static_cast<int64_t>(b) * D + c] : 0.f;
  for (int lot = 0; lot < lots; ++lot) {
    asm volatile("cp.async.wait_group %0;" ::"n"(FOLD_STAGES - 2) : "memory");
    __syncthreads();                             // this lot is in, and the first warp is done with the last one, whose place is asked for
    request(lot + FOLD_STAGES - 1);
    if (warp == 0 && active) {
      const FoldStage& s = stages[lot % FOLD_STAGES];
      const int n = min(FOLD_TILES, tiles - lot * FOLD_TILES);
      const float first = state;
      float* const from = out;
      uint32_t largest = 0u;                     // of the factors' bits: plain ones are below infinity's
      int i = 0;
      for (; i + 8 <= n; i += 8) {               // eight maps in registers at a time, so that the walk waits for its own sums only
        float a[8], h[8];
        int cuts = 0;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          a[k] = s.A[i + k][lane];
          h[k] = s.H[i + k][lane];
          if (cut) cuts |= (s.cut[i + k] != 0) << k;
          largest = max(largest, __float_as_uint(a[k]));
        }
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          *out = state;
          out += step;
          state = cuts >> k & 1 ? h[k] : fmaf(a[k], state, h[k]);
        }
      }
      for (; i < n; ++i) {
        *out = state;
        out += step;
        largest = max(largest, __float_as_uint(s.A[i][lane]));
        state = cut && s.cut[i] ? s.H[i][lane] : fmaf(s.A[i][lane], state, s.H[i][lane]);
      }
      if (largest >= 0x7f800000u) {              // once more for factors out of range (tgdn_scan.cuh); a test every eight maps took a third longer
        state = first;
        out = from;
#pragma unroll 1
        for (i = 0; i < n; ++i) {
          *out = state;
          out += step;
          state = cut && s.cut[i] ? s.H[i][lane] : factor_apply(s.A[i][lane], state, s.H[i][lane]);
        }
      }
    }
  }
  if (end && warp == 0 && active) end[static_cast<int64_t>(b) * D + c] = state;
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

// The way over the tiles, by the size of the problem alone.  One block walks a tile in 1.3 us forward and 2 us backward, whatever the slices
// beside it (bf16, up to one block an SM); the split way's three launches begin at 9 and 11 us and its two passes over the data add 0.015 and
// 0.019 us a tile and slice.  So the split way is ahead from 6 tiles on for one slice (64 channels x 16384: 163 -> 11 us forward), from 17 for
// 64 slices (4096 channels x 4096: 44 -> 36 us, x 1024: 12 -> 13 us), and not above 90 (6144 x 4096: 45 and 59 us).  Four more launches of a
// forward and backward cost the host 15 us where it is what a call waits for (3 x 1000 x 333: 69 and 84 us a step): twice the tiles.
// Slices are counted as 64 channels for every kernel, as the measurements are; kernels of single channels have twice the blocks.
bool scan_splits(int B, int T, int D) {
  const int64_t units = static_cast<int64_t>(B) * ((D + 63) / 64), tiles = (T - 1) / SCAN_TILE + 1, spare = tgdn_sm_count() * 5 / 8 - units;
  return spare > 0 && tiles * spare > 1000;
}
// Blocks of the two passes: a few tiles each, enough of them for four rounds over the SMs.
void scan_spans(ScanParams& p) {
  const int64_t units = static_cast<int64_t>(p.B) * ((p.D + 63) / 64), all = units * p.tiles;
  int64_t per = (all + 4 * tgdn_sm_count() - 1) / (4 * tgdn_sm_count());
  if (per < 2) per = 2;
  p.per_span = static_cast<int>(per);
  p.spans = (p.tiles + p.per_span - 1) / p.per_span;
}
int scan_fold(const ScanParams& p, bool reverse, const float* start, float* carry, float* end, cudaStream_t s) {
  static bool configured[2][64] = {};
  constexpr int bytes = FOLD_STAGES * sizeof(FoldStage);
  const int64_t blocks = static_cast<int64_t>(p.B) * ((p.D + 31) / 32);
  const void* kernel = reverse ? reinterpret_cast<const void*>(scan_fold_kernel<true>) : reinterpret_cast<const void*>(scan_fold_kernel<false>);
  if (const int rc = tgdn_dynamic_smem(kernel, bytes, configured[reverse])) return rc;
  if (reverse) scan_fold_kernel<true><<<static_cast<unsigned>(blocks), FOLD_THREADS, bytes, s>>>(p.map_a, p.map_h, p.map_cut, start, carry, end, p.tiles, p.D);
  else scan_fold_kernel<false><<<static_cast<unsigned>(blocks), FOLD_THREADS, bytes, s>>>(p.map_a, p.map_h, p.map_cut, start, carry, end, p.tiles, p.D);
  return tgdn_cuda_error(cudaGetLastError());
}

ScanIn scan_in(const tgdn_rows& t, int T) { return {t.data, t.stride_outer, T == 1 ? 0 : static_cast<int>(t.stride_inner)}; }

// What the copy engine takes: rows of whole 16-byte pieces that follow one another.  Pairs of the outputs follow from D.
bool in_pieces(const tgdn_rows& t, int B, int T, int D) {
  const int64_t piece = 16 / type_bytes(t.type);
  return reinterpret_cast<uintptr_t>(t.data) % 16 == 0 && D % piece == 0 && (T == 1 || (t.stride_inner >= D && t.stride_inner % piece == 0)) &&
         (B == 1 || (t.stride_outer > 0 && t.stride_outer % piece == 0 && t.stride_outer < int64_t{1} << 36));
}
bool aligned(const void* p, int bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

int scan_checks(const tgdn_rows* x, const tgdn_rows* g, const int32_t* map, int n_docs, int B, int T, int D) {
  if (!x || !g || !x->data || !g->data) return TGDN_ERR_NULL;
  if (B <= 0 || T <= 0 || T > 0x7fffffff - 2 * SCAN_TILE || D <= 0 || D > 0x7fffffff - 64 || (map && (B != 1 || n_docs <= 0))) return TGDN_ERR_SHAPE;
  if (!type_known(x->type) || !type_known(g->type)) return TGDN_ERR_TYPE;
  if (x->stride_inner > 0x7fffffffLL || g->stride_inner > 0x7fffffffLL || x->stride_inner < 0 || g->stride_inner < 0) return TGDN_ERR_SHAPE;
  return 0;
}

}  // namespace

extern "C" int64_t tgdn_scan_carry_floats(int B, int T, int D) {
  return static_cast<int64_t>(B) * ((T + static_cast<int64_t>(SCAN_TILE) - 1) / SCAN_TILE) * D;
}

// The tiles' maps (two numbers a tile and channel), the states between the tiles, and where documents' borders lie.
extern "C" int64_t tgdn_scan_scratch_floats(int B, int T, int D) {
  if (B <= 0 || T <= 0 || D <= 0 || !scan_splits(B, T, D)) return 0;
  return 3 * tgdn_scan_carry_floats(B, T, D) + (T - 1) / SCAN_TILE + 1;
}

extern "C" int tgdn_scan_map(const void* cu_seqlens, int cu_is_int64, int n_docs, int T, int32_t* map, uint8_t* valid, void* stream) {
  if (!cu_seqlens || !map || !valid) return TGDN_ERR_NULL;
  if (n_docs <= 0 || T <= 0) return TGDN_ERR_SHAPE;
  if (!tgdn_check_device()) return TGDN_ERR_DEVICE;
  scan_map_kernel<<<T / 256 + (T % 256 != 0), 256, 0, static_cast<cudaStream_t>(stream)>>>(cu_seqlens, cu_is_int64, n_docs, T, map, valid);
  return tgdn_cuda_error(cudaGetLastError());
}

extern "C" int tgdn_scan_fwd(const tgdn_rows* host_x, const tgdn_rows* host_g, const int32_t* map, int n_docs, int B, int T, int D,
                             const float* initial, void* h, float* final_state, float* carry, float* scratch, int64_t scratch_floats,
                             void* stream) {
  if (const int rc = scan_checks(host_x, host_g, map, n_docs, B, T, D)) return rc;
  if (!h) return TGDN_ERR_NULL;
  const int64_t needed = tgdn_scan_scratch_floats(B, T, D), states = tgdn_scan_carry_floats(B, T, D);
  if (needed > 0 && (!scratch || scratch_floats < needed)) return TGDN_ERR_SCRATCH;
  if (!tgdn_check_device()) return TGDN_ERR_DEVICE;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  ScanParams p{};
  p.x = scan_in(*host_x, T);
  p.g = scan_in(*host_g, T);
  p.map = map; p.initial = initial; p.h = h; p.final_state = final_state; p.carry = carry;
  p.B = B; p.T = T; p.D = D; p.n_docs = n_docs;
  p.tiles = p.per_span = (T - 1) / SCAN_TILE + 1;
  p.spans = 1;
  p.status = tgdn_status_word();
  const bool pieces = in_pieces(*host_x, B, T, D) && in_pieces(*host_g, B, T, D) && aligned(h, 8);
  const int xt = host_x->type, gt = host_g->type;
  if (needed == 0) return tgdn_scan_launch_fwd(p, xt, gt, pieces, SCAN_WHOLE, s);
  scan_spans(p);
  p.map_a = scratch; p.map_h = scratch + states;
  if (!p.carry) p.carry = scratch + 2 * states;
  if (map) p.map_cut = reinterpret_cast<int*>(scratch + 3 * states);
  if (const int rc = tgdn_scan_launch_fwd(p, xt, gt, pieces, SCAN_MAPS, s)) return rc;
  if (const int rc = scan_fold(p, false, map ? nullptr : initial, p.carry, map ? nullptr : final_state, s)) return rc;
  return tgdn_scan_launch_fwd(p, xt, gt, pieces, SCAN_FINISH, s);
}

extern "C" int tgdn_scan_bwd(const tgdn_rows* host_x, const tgdn_rows* host_g, const tgdn_rows* host_dh, const int32_t* map, int n_docs,
                             int B, int T, int D, const float* initial, const float* carry, const float* dfinal, void* dx, void* dg,
                             float* dinitial, float* scratch, int64_t scratch_floats, void* stream) {
  if (const int rc = scan_checks(host_x, host_g, map, n_docs, B, T, D)) return rc;
  if (!host_dh || !host_dh->data || !carry || !dx || !dg) return TGDN_ERR_NULL;
  if (host_dh->type != host_x->type) return TGDN_ERR_TYPE;
  if (host_dh->stride_inner > 0x7fffffffLL || host_dh->stride_inner < 0) return TGDN_ERR_SHAPE;
  const int64_t needed = tgdn_scan_scratch_floats(B, T, D), states = tgdn_scan_carry_floats(B, T, D);
  if (needed > 0 && (!scratch || scratch_floats < needed)) return TGDN_ERR_SCRATCH;
  if (!tgdn_check_device()) return TGDN_ERR_DEVICE;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  ScanParams p{};
  p.x = scan_in(*host_x, T);
  p.g = scan_in(*host_g, T);
  p.dh = scan_in(*host_dh, T);
  p.map = map; p.initial = initial; p.carry = const_cast<float*>(carry); p.dfinal = dfinal;
  p.dx = dx; p.dg = dg; p.dinitial = dinitial;
  p.B = B; p.T = T; p.D = D; p.n_docs = n_docs;
  p.tiles = p.per_span = (T - 1) / SCAN_TILE + 1;
  p.spans = 1;
  p.status = tgdn_status_word();
  const bool pieces = in_pieces(*host_x, B, T, D) && in_pieces(*host_g, B, T, D) && in_pieces(*host_dh, B, T, D) && aligned(dx, 8) && aligned(dg, 8);
  const int xt = host_x->type, gt = host_g->type;
  if (needed == 0) return tgdn_scan_launch_bwd(p, xt, gt, pieces, SCAN_WHOLE, s);
  scan_spans(p);
  p.map_a = scratch; p.map_h = scratch + states; p.mu = scratch + 2 * states;
  if (map) p.map_cut = reinterpret_cast<int*>(scratch + 3 * states);
  if (const int rc = tgdn_scan_launch_bwd(p, xt, gt, pieces, SCAN_MAPS, s)) return rc;
  if (const int rc = scan_fold(p, true, map ? nullptr : dfinal, p.mu, map ? nullptr : dinitial, s)) return rc;
  return tgdn_scan_launch_bwd(p, xt, gt, pieces, SCAN_FINISH, s);
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
