// C ABI of the operators between and beside the packed linears of a transformer block: rotary
// positions, attention over packed sequences, the dense 16-bit linear.
#include <algorithm>
#include <atomic>
#include <climits>
#include <cmath>

#include "../../include/oc_b200.h"
#include "common.cuh"
#include "host.h"
#include "rope.cuh"
#include "attn_common.cuh"
#include "attn_split.cuh"
#include "attn_tile.cuh"
#include "gemm_dense.cuh"

// This translation unit's device error word (common.cuh defines one per unit), for
// oc_b200_read_device_error.
int block_ops_device_error(unsigned* value, cudaStream_t stream) {
  const unsigned zero = 0;
  if (int rc = cuda_check(cudaMemcpyFromSymbolAsync(value, oc::g_oc_dev_error, sizeof(*value), 0,
                                                    cudaMemcpyDeviceToHost, stream), "read device error"))
    return rc;
  return cuda_check(cudaMemcpyToSymbolAsync(oc::g_oc_dev_error, &zero, sizeof(zero), 0, cudaMemcpyHostToDevice, stream),
                    "clear device error");
}

namespace {

// Raises a kernel's dynamic shared memory limit, an attribute per device: set once on each, remembered in
// the launcher's own word.
template <typename K> int set_smem(K kern, int bytes, std::atomic<uint64_t>& done) {
  int dev = 0;
  if (int rc = current_device(&dev)) return rc;
  const uint64_t bit = dev < 64 ? 1ull << dev : 0;
  if (bit & done.load(std::memory_order_relaxed)) return OC_OK;
  if (int rc = cuda_check(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes),
                          "shared memory limit"))
    return rc;
  done.fetch_or(bit, std::memory_order_relaxed);
  return OC_OK;
}

// A kernel that moves registers between its warpgroups (setmaxnreg) waits for ever if the launch gives it
// fewer than the shares add up to, so the compiled count is checked before the first launch.
template <typename K> int check_registers(K kern, int threads, int needed, const char* what) {
  cudaFuncAttributes at;
  if (int rc = cuda_check(cudaFuncGetAttributes(&at, kern), what)) return rc;
  if (at.numRegs * threads < needed)
    return fail(OC_ERR_UNSUPPORTED, "%s: built with %d registers a thread, %d threads need %d in all", what, at.numRegs,
                threads, needed);
  return OC_OK;
}

// Rows, sequences, heads and features stay below 2^30, so that sums of two of them, and the last block of keys
// or tile of rows that begins below a count, stay below 2^31.
bool too_many(int n) { return n >= 1 << 30; }

// ------------------------------------------------------------------ rotary positions
template <int DT, int V, bool INTER>
int launch_rope(const oc::RopeParams& p0, int sms, cudaStream_t stream) {
  oc::RopeParams p = p0;
  const long long heads = (long long)p.t[0].H + p.t[1].H;
  // Four tokens to a block once that still gives every SM several blocks; below, one token, its heads
  // spread over blocks until about two blocks per SM run.
  const int tb = p.T >= 4 * 4 * sms ? 4 : 1;
  const long long gx = ((long long)p.T + tb - 1) / tb;
  long long want = gx >= 2 * sms ? 1 : (2 * sms + gx - 1) / gx;
  if (want > heads) want = heads;
  p.heads_per_block = (int)((heads + want - 1) / want);
  const dim3 grid((unsigned)gx, (unsigned)((heads + p.heads_per_block - 1) / p.heads_per_block));
  const size_t smem = (size_t)tb * p.R * sizeof(float);
  if (tb == 4)
    oc::rope_kernel<DT, V, INTER, 4><<<grid, oc::kRopeThreads, smem, stream>>>(p);
  else
    oc::rope_kernel<DT, V, INTER, 1><<<grid, oc::kRopeThreads, smem, stream>>>(p);
  return launch_check("rope");
}

template <int DT, int VMAX>
int launch_rope_dt(const oc::RopeParams& p, bool vec, bool inter, int sms, cudaStream_t stream) {
  if (vec) return inter ? launch_rope<DT, VMAX, true>(p, sms, stream) : launch_rope<DT, VMAX, false>(p, sms, stream);
  return inter ? launch_rope<DT, 1, true>(p, sms, stream) : launch_rope<DT, 1, false>(p, sms, stream);
}

// ------------------------------------------------------------------ attention
int attn_dp(int D) { return D <= 64 ? 64 : D <= 128 ? 128 : 256; }

template <int DP> int split_ctas(int sms) { return sms * oc::SplitCfg<DP>::kCtasPerSm; }
int split_ctas(int dp, int sms) {
  return dp == 64 ? split_ctas<64>(sms) : dp == 128 ? split_ctas<128>(sms) : split_ctas<256>(sms);
}
size_t split_desc_bytes(int ctas) { return (((size_t)ctas * oc::kSplitDescInts * 4) + 255) / 256 * 256; }
size_t split_ws_bytes(int dp, int ctas) {
  return split_desc_bytes(ctas) + (size_t)ctas * 2 * oc::kSplitRows * (dp + 2) * 4;
}

// Which kernel a call takes, and its workspace. The host knows the longest query run (max_q) or, without
// it, the mean one.
constexpr int kTileMinRows = 16;
struct AttnPlan {
  bool tile;
  int dp, ctas;      // split kernel: its grid
  oc::TileGrid tg;
  size_t ws;
};

AttnPlan attn_plan(int Tq, int Tk, int B, int Hq, int Hkv, int D, int max_q, int sms) {
  AttnPlan pl{};
  pl.dp = attn_dp(D);
  const int64_t seqs = std::max(B, 1), G = Hq / Hkv;
  const int64_t run = max_q > 0 ? std::min(max_q, Tq) : (Tq + seqs - 1) / seqs;
  // One tile of 16 (token, head) rows streams the keys from memory at the split kernel's rate; more rows read them
  // again there and are tensor work here. 16 sequences of 2048 to 4096 keys in a graph, tile against split kernel:
  // heads of 128, 32 rows 65.4 and 58.9 us, 48 rows 63.9 and 72.9, 64 rows 65.4 and 112; heads of 64, 32 rows 95.4 and
  // 87.6, 64 rows 88.0 and 131; heads of 256, 18 rows 57.0 and 62.5, 36 rows 59.2 and 75.2.
  pl.tile = run * G > kTileMinRows && G <= 128 && B > 0 && Tk > 0;
  if (!pl.tile) {
    pl.ctas = split_ctas(pl.dp, sms);
    pl.ws = split_ws_bytes(pl.dp, pl.ctas);
    return pl;
  }
  const int tiles = pl.dp == 256 ? 1 : 2;
  pl.tg.tokens = 128 / (int)G;
  const int64_t range = (int64_t)tiles * pl.tg.tokens;
  pl.tg.slots = (int)(Tq / range) + B;
  // Ranges that hold tokens, about; with fewer of them than SMs the keys of each are split over several
  // CTAs, at least two blocks of keys to a part.
  const int64_t busy = Hkv * std::max(seqs * ((run + range - 1) / range), Tq / range);
  const int64_t blocks = ((Tk + seqs - 1) / seqs + oc::kTileKeys - 1) / oc::kTileKeys;
  pl.tg.splits = (int)std::max<int64_t>(1, std::min<int64_t>({sms / busy, blocks / 2, 32}));
  if (pl.tg.splits > 1)
    pl.ws = (size_t)pl.tg.slots * Hkv * pl.tg.splits * tiles * 128 * (pl.dp + 2) * 4;
  return pl;
}

template <bool BF16, int DP> int launch_split(const oc::AttnParams& p, int ctas, cudaStream_t stream) {
  auto kern = oc::attn_split_kernel<BF16, DP>;
  static std::atomic<uint64_t> smem_set{0};
  if (int rc = set_smem(kern, oc::SplitCfg<DP>::kRingBytes, smem_set)) return rc;
  kern<<<ctas, oc::SplitCfg<DP>::kThreads, oc::SplitCfg<DP>::kRingBytes, stream>>>(p);
  if (int rc = launch_check("attention (split)")) return rc;
  return launch_pdl(oc::attn_join_kernel<BF16, DP>, dim3((unsigned)ctas, oc::kSplitRows / 4), dim3(oc::kJoinThreads), 0,
                    stream,
                    "attention (join)", p);
}

// [rows, heads, D] tensor in boxes of `rows` rows x `heads` heads x 64 columns. A dimension of one row or
// head takes any valid stride.
int attn_tmap(CUtensorMap* map, bool bf16, const void* base, int D, int H, int T, int64_t sh, int64_t st, int heads,
              int rows) {
  EncodeTiledFn fn = encode_fn();
  if (!fn) return fail(OC_ERR_CUDA, "cuTensorMapEncodeTiled entry point unavailable");
  cuuint64_t dims[3] = {(cuuint64_t)D, (cuuint64_t)H, (cuuint64_t)T};
  cuuint64_t strides[2] = {(cuuint64_t)(H > 1 ? sh : D) * 2, (cuuint64_t)(T > 1 ? st : D) * 2};
  cuuint32_t box[3] = {64, (cuuint32_t)heads, (cuuint32_t)rows}, estr[3] = {1, 1, 1};
  const CUresult r = fn(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3,
                        const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                        CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(OC_ERR_CUDA, "attention: cuTensorMapEncodeTiled failed (%d)", (int)r);
  return OC_OK;
}

template <bool BF16, int DP> int launch_tile(oc::AttnParams p, const oc::TileGrid& tg, cudaStream_t stream) {
  using Cfg = oc::TileCfg<DP>;
  oc::TileMaps maps;
  if (int rc = attn_tmap(&maps.q, BF16, p.q, p.D, p.Hq, p.Tq, p.q_sh, p.q_st, p.G, tg.tokens)) return rc;
  if (int rc = attn_tmap(&maps.k, BF16, p.k, p.D, p.Hkv, p.Tk, p.k_sh, p.k_st, 1, oc::kTileKeys)) return rc;
  if (int rc = attn_tmap(&maps.v, BF16, p.v, p.D, p.Hkv, p.Tk, p.v_sh, p.v_st, 1, oc::kTileKeys)) return rc;
  const long long units = (long long)tg.slots * p.Hkv;
  if (units * tg.splits > INT_MAX / 2) return fail(OC_ERR_INVALID, "attention: %lld token ranges", units);
  // The softmax takes its maximum before the scale: a negative scale negates Q in the product. A scale of
  // zero makes every finite score zero there and every other NaN, and a scale of one keeps them so.
  const int mode = (p.scale_log2 < 0.f ? oc::kTileNegate : 0) | (p.scale_log2 == 0.f ? oc::kTileZeroScale : 0);
  p.scale_log2 = mode & oc::kTileZeroScale ? 1.f : std::fabs(p.scale_log2);
  auto kern = oc::attn_tile_kernel<BF16, DP>;
  static const int regs_rc = check_registers(
      kern, Cfg::kThreads, Cfg::kTiles == 2 ? Cfg::kSoftmaxThreads * Cfg::kSoftmaxRegs + 128 * Cfg::kAuxRegs : 0,
      "attention (tile)");
  if (regs_rc) return fail(regs_rc, "attention (tile): register count of the build");
  static std::atomic<uint64_t> smem_set{0};
  if (int rc = set_smem(kern, Cfg::kSmem, smem_set)) return rc;
  kern<<<(unsigned)(units * tg.splits), Cfg::kThreads, Cfg::kSmem, stream>>>(maps, p, tg, mode);
  if (int rc = launch_check("attention (tile)")) return rc;
  if (tg.splits == 1) return OC_OK;
  // the tile kernel gives no signal, yet this launch starts 0.7 us earlier than a plain one (7 x 5 tokens, heads of 256)
  return launch_pdl(oc::attn_tile_join_kernel<BF16, DP>, dim3((unsigned)(units * Cfg::kTiles), 4, DP / 64), dim3(256), 0, stream,
                    "attention (tile join)", p, tg);
}

// ------------------------------------------------------------------ dense linear
template <bool BF16, int BN>
int launch_dense_split(const void* x, int64_t ldx, const void* w, int64_t ldw, oc::DenseParams p, int dev,
                       cudaStream_t stream) {
  using Cfg = oc::DsCfg<BN>;
  const CUtensorMapDataType dt = BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  CUtensorMap tw, tx;
  if (int rc = make_tmap_2d(&tw, dt, 2, w, p.K, p.N, (uint64_t)ldw * 2, 64, 128, CU_TENSOR_MAP_SWIZZLE_128B)) return rc;
  if (int rc = make_tmap_2d(&tx, dt, 2, x, p.K, p.M, (uint64_t)ldx * 2, 64, BN, CU_TENSOR_MAP_SWIZZLE_128B)) return rc;
  p.n_tiles_m = (p.M + BN - 1) / BN;
  const long long tiles = (long long)((p.N + 127) / 128) * p.n_tiles_m;
  const int slots = sm_count(dev) * (BN <= 64 ? 2 : 1);
  const int kb = (p.K + 63) / 64;
  int S = 1;
  while (S < 8 && tiles * S * 2 <= slots && kb >= S * 2 * 2) S *= 2;
  if (tiles * S > INT_MAX) return fail(OC_ERR_INVALID, "dense_gemm: %lld tiles", tiles);
  auto kern = oc::dense_split_kernel<BF16, BN>;
  static std::atomic<uint64_t> smem_set{0};
  if (int rc = set_smem(kern, Cfg::kSmem, smem_set)) return rc;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(tiles * S));
  cfg.blockDim = dim3(oc::kDsThreads);
  cfg.dynamicSmemBytes = Cfg::kSmem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = S;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (int rc = cuda_check(cudaLaunchKernelEx(&cfg, kern, tw, tx, p), "dense_gemm")) return rc;
  return launch_check("dense_gemm");
}

// Tokens of a tile of the K-splitting kernel, or 0 where the pairs take the call.
// The K-splitting kernel up to 32 tokens, where streaming the weights through every SM decides (one token,
// weights from HBM, 4096 x 4096: 12.8 us against 16.8 of the pairs; 1024 x 8192: 10.8 against 27.1). Above, the
// pairs (64 tokens, weights in L2: 2560 x 2560 8.5 us against 13.2, 4096 x 4096 11.0 against 15.7), unless few of them
// would walk a long K (64 tokens, 1024 x 8192 from HBM: 13.8 against 26.9; 128 tokens: 16.2 against 25.1). In between
// neither wins everywhere (4096 x 8192, pairs and split: 33 tokens 17.0 and 15.1, 64 tokens 17.3 and 18.7, 128 tokens
// 22.6 and 18.0).
int dense_split_tokens(int M, int N, int K) {
  const int least_tiles = (N + 255) / 256 * ((M + 31) / 32);   // of the pairs, at 32 tokens each
  if (M <= 16) return 16;
  if (M <= 32) return 32;
  if (M <= 128 && least_tiles <= 24 && K > 4096) return M <= 64 ? 64 : 128;
  return 0;
}

// Tokens of a tile for the pair kernel: equal tiles of a multiple of 32 tokens, the size with the least
// (waves of CTA pairs) x (time of one tile). A 64-k step of a tile takes about 2.3 cycles per token
// (measured 590 at 256 tokens, 295 at 128), but no less than about 250, where the weights' stream bounds
// it; a wave costs about 2500 cycles besides. Measured on 256 x 4096 x 4096: tiles of 256, 128, 64, 32 tokens
// take 25.1, 18.3, 17.5 and 24.0 us; on 256 x 12288 x 4096: 28.7, 35.6, 42.1 and 55.0 us.
int dense_bt(int M, int tiles_n, int K, int pairs) {
  const int kb = (K + 63) / 64;
  int best = 256;
  double best_cost = 1e300;
  for (int want = 256; want >= 64; want -= 32) {   // below 64 a tile takes no less time
    const int tiles_m = (M + want - 1) / want;
    const int bt = ((M + tiles_m - 1) / tiles_m + 31) / 32 * 32;
    const double waves = std::ceil((double)tiles_n * tiles_m / pairs);
    const double cost = waves * (kb * std::max(250.0, 2.3 * bt) + 2500.0);
    if (cost < best_cost) {
      best_cost = cost;
      best = bt;
    }
  }
  return best;
}

template <bool BF16, int ACT, bool RES>
int launch_dense_tile(const void* x, int64_t ldx, const void* w, int64_t ldw, const oc::DenseParams& d, int dev,
                      cudaStream_t stream) {
  const CUtensorMapDataType dt = BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  oc::DenseTileParams p{};
  p.d = d;
  const int max_pairs = sm_count(dev) / 2;
  p.tiles_n = (d.N + 255) / 256;
  p.bt = dense_bt(d.M, p.tiles_n, d.K, max_pairs);
  p.tiles_m = (d.M + p.bt - 1) / p.bt;
  const long long tiles = (long long)p.tiles_n * p.tiles_m;
  if (tiles > INT_MAX / 2) return fail(OC_ERR_INVALID, "dense_gemm: %lld tiles", tiles);
  p.tiles = (int)tiles;
  p.tma_epi = d.vec;
  CUtensorMap tw, tx, tc = {}, tr = {};
  if (int rc = make_tmap_2d(&tw, dt, 2, w, d.K, d.N, (uint64_t)ldw * 2, 64, 128, CU_TENSOR_MAP_SWIZZLE_128B)) return rc;
  if (int rc = make_tmap_2d(&tx, dt, 2, x, d.K, d.M, (uint64_t)ldx * 2, 64, p.bt / 2, CU_TENSOR_MAP_SWIZZLE_128B))
    return rc;
  if (p.tma_epi) {
    if (int rc = make_tmap_2d(&tc, dt, 2, d.out, d.N, d.M, (uint64_t)d.ldc * 2, 32, 32, CU_TENSOR_MAP_SWIZZLE_NONE)) return rc;
    if (RES)
      if (int rc = make_tmap_2d(&tr, dt, 2, d.residual, d.N, d.M, (uint64_t)d.ldr * 2, 32, 32, CU_TENSOR_MAP_SWIZZLE_NONE))
        return rc;
  }
  auto kern = oc::dense_tile_kernel<BF16, ACT, RES>;
  static std::atomic<uint64_t> smem_set{0};
  if (int rc = set_smem(kern, oc::kDtSmem, smem_set)) return rc;
  const int pairs = (int)std::min<long long>(tiles, max_pairs);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(2 * pairs));
  cfg.blockDim = dim3(oc::kDtThreads);
  cfg.dynamicSmemBytes = oc::kDtSmem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 2;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (int rc = cuda_check(cudaLaunchKernelEx(&cfg, kern, tw, tx, tc, tr, p), "dense_gemm (pairs)")) return rc;
  return launch_check("dense_gemm (pairs)");
}

template <bool BF16, bool RES>
int launch_dense_tile_act(const void* x, int64_t ldx, const void* w, int64_t ldw, const oc::DenseParams& p, int dev,
                          cudaStream_t stream) {
  switch (p.act) {
    case OC_ACT_GELU_TANH: return launch_dense_tile<BF16, oc::kDenseGeluTanh, RES>(x, ldx, w, ldw, p, dev, stream);
    case OC_ACT_GELU: return launch_dense_tile<BF16, oc::kDenseGelu, RES>(x, ldx, w, ldw, p, dev, stream);
    case OC_ACT_SILU: return launch_dense_tile<BF16, oc::kDenseSilu, RES>(x, ldx, w, ldw, p, dev, stream);
    case OC_ACT_RELU: return launch_dense_tile<BF16, oc::kDenseRelu, RES>(x, ldx, w, ldw, p, dev, stream);
    default: return launch_dense_tile<BF16, oc::kDenseNone, RES>(x, ldx, w, ldw, p, dev, stream);
  }
}

template <bool BF16>
int launch_dense(const void* x, int64_t ldx, const void* w, int64_t ldw, const oc::DenseParams& p, int dev,
                 cudaStream_t stream) {
  const int split = dense_split_tokens(p.M, p.N, p.K);
  if (split == 16) return launch_dense_split<BF16, 16>(x, ldx, w, ldw, p, dev, stream);
  if (split == 32) return launch_dense_split<BF16, 32>(x, ldx, w, ldw, p, dev, stream);
  if (split == 64) return launch_dense_split<BF16, 64>(x, ldx, w, ldw, p, dev, stream);
  if (split == 128) return launch_dense_split<BF16, 128>(x, ldx, w, ldw, p, dev, stream);
  return p.residual ? launch_dense_tile_act<BF16, true>(x, ldx, w, ldw, p, dev, stream)
                    : launch_dense_tile_act<BF16, false>(x, ldx, w, ldw, p, dev, stream);
}

}  // namespace

extern "C" int oc_b200_rope(const void* q, int64_t q_st, int64_t q_sh, void* q_out, int64_t qo_st, int64_t qo_sh,
                            int Hq, const void* k, int64_t k_st, int64_t k_sh, void* k_out, int64_t ko_st,
                            int64_t ko_sh, int Hk, int dtype, int T, int D, int R, const void* positions,
                            int positions_64, int64_t positions_st, const uint64_t* turns, const uint8_t* axis,
                            float gain, int interleaved, oc_stream_t stream_) {
  if (T < 0 || Hq < 0 || Hk < 0 || D <= 0 || D > 1024 || R <= 0 || R > D || R % 2 != 0)
    return fail(OC_ERR_INVALID, "rope: T=%d Hq=%d Hk=%d D=%d R=%d (R even, at most D; D at most 1024)", T, Hq, Hk, D, R);
  if (!dtf(dtype)) return fail(OC_ERR_INVALID, "rope: dtype %d", dtype);
  if (too_many(T) || too_many(Hq) || too_many(Hk))
    return fail(OC_ERR_INVALID, "rope: T=%d Hq=%d Hk=%d (below 2^30)", T, Hq, Hk);
  if (T == 0 || Hq + Hk == 0) return OC_OK;
  if ((Hq && (!q || !q_out)) || (Hk && (!k || !k_out)) || !positions || !turns)
    return fail(OC_ERR_INVALID, "rope: NULL pointer");
  if (!std::isfinite(gain)) return fail(OC_ERR_INVALID, "rope: gain %g", (double)gain);
  oc::RopeParams p{};
  p.t[0] = {q, q_out, q_st, q_sh, qo_st, qo_sh, Hq};
  p.t[1] = {k, k_out, k_st, k_sh, ko_st, ko_sh, Hk};
  p.T = T;
  p.D = D;
  p.R = R;
  p.pos = positions;
  p.pos64 = positions_64;
  p.pos_st = positions_st;
  p.turns = reinterpret_cast<const unsigned long long*>(turns);
  p.axis = axis;
  p.gain = gain;
  p.copy_rest = D > R && ((Hq && q != q_out) || (Hk && k != k_out));
  const int v = dtype == OC_DT_F32 ? 4 : 8;
  bool vec = D % (2 * v) == 0 && R % (2 * v) == 0;
  for (const oc::RopeTensor& t : p.t)
    if (t.H && (!aligned(t.x, 16) || !aligned(t.y, 16) || t.xst % v || t.xsh % v || t.yst % v || t.ysh % v)) vec = false;
  // without vectors the copied part moves in units of two values
  if (!vec && p.copy_rest && (D - R) % 2 != 0)
    return fail(OC_ERR_INVALID, "rope: D=%d must be even out of place", D);
  int dev = 0;
  if (int rc = current_device(&dev)) return rc;
  const int sms = sm_count(dev);
  cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_);
  if (dtype == OC_DT_F16) return launch_rope_dt<oc::kF16, 8>(p, vec, interleaved != 0, sms, stream);
  if (dtype == OC_DT_BF16) return launch_rope_dt<oc::kBF16, 8>(p, vec, interleaved != 0, sms, stream);
  return launch_rope_dt<oc::kF32, 4>(p, vec, interleaved != 0, sms, stream);
}

extern "C" size_t oc_b200_attention_workspace(int Tq, int Tk, int B, int Hq, int Hkv, int D, int max_q) {
  if (Tq <= 0 || Tk < 0 || B < 0 || Hq <= 0 || Hkv <= 0 || Hq % Hkv != 0 || D <= 0 || D > 256) return 0;
  if (too_many(Tq) || too_many(Tk) || too_many(B) || too_many(Hq)) return 0;
  int dev = 0;
  if (current_device(&dev)) return 0;
  return attn_plan(Tq, Tk, B, Hq, Hkv, D, max_q, sm_count(dev)).ws;
}

extern "C" int oc_b200_attention(const void* q, int64_t q_st, int64_t q_sh, const void* k, int64_t k_st, int64_t k_sh,
                                 const void* v, int64_t v_st, int64_t v_sh, void* out, int64_t o_st, int64_t o_sh,
                                 int dtype, int Tq, int Tk, int Hq, int Hkv, int D, const int32_t* cu_q,
                                 const int32_t* cu_k, const int32_t* kv_lens, int B, int causal, float scale,
                                 int max_q, int zero_unowned, void* workspace, size_t workspace_bytes,
                                 oc_stream_t stream_) {
  if (!dt16(dtype)) return fail(OC_ERR_INVALID, "attention: dtype %d (f16 or bf16)", dtype);
  if (Tq < 0 || Tk < 0 || B < 0 || Hq <= 0 || Hkv <= 0 || Hq % Hkv != 0)
    return fail(OC_ERR_INVALID, "attention: Tq=%d Tk=%d B=%d Hq=%d Hkv=%d (Hq a multiple of Hkv)", Tq, Tk, B, Hq, Hkv);
  if (D <= 0 || D > 256 || D % 8 != 0)
    return fail(OC_ERR_UNSUPPORTED, "attention: head size %d (a multiple of 8 up to 256)", D);
  if (too_many(Tq) || too_many(Tk) || too_many(B) || too_many(Hq))
    return fail(OC_ERR_INVALID, "attention: Tq=%d Tk=%d B=%d Hq=%d (below 2^30)", Tq, Tk, B, Hq);
  if ((cu_q == nullptr) != (cu_k == nullptr)) return fail(OC_ERR_INVALID, "attention: cu_q and cu_k come together");
  if (!cu_q && B != 1) return fail(OC_ERR_INVALID, "attention: B=%d without sequence tables", B);
  if (!std::isfinite(scale * 1.4426950408889634f)) return fail(OC_ERR_INVALID, "attention: scale %g", (double)scale);
  if (Tq == 0 || (B == 0 && !zero_unowned)) return OC_OK;
  if (!q || !out || (Tk > 0 && (!k || !v))) return fail(OC_ERR_INVALID, "attention: NULL pointer");
  const void* ptrs[4] = {q, Tk > 0 ? k : q, Tk > 0 ? v : q, out};
  const int64_t strides[8] = {q_st, q_sh, k_st, k_sh, v_st, v_sh, o_st, o_sh};
  for (const void* ptr : ptrs)
    if (!aligned(ptr, 16)) return fail(OC_ERR_INVALID, "attention: tensors must be 16-byte aligned");
  for (int64_t st : strides)
    if (st % 8 != 0 || st < 0)
      return fail(OC_ERR_INVALID, "attention: stride %lld (a multiple of 8 elements)", (long long)st);
  int dev = 0;
  if (int rc = current_device(&dev)) return rc;
  AttnPlan pl = attn_plan(Tq, Tk, B, Hq, Hkv, D, max_q, sm_count(dev));
  if (pl.ws && (!workspace || workspace_bytes < pl.ws || !aligned(workspace, 16)))
    return fail(OC_ERR_WORKSPACE, "attention: needs %zu bytes of 16-byte aligned workspace, got %zu", pl.ws,
                workspace_bytes);
  oc::AttnParams p{};
  p.q = reinterpret_cast<const uint16_t*>(q);
  p.k = reinterpret_cast<const uint16_t*>(Tk > 0 ? k : q);
  p.v = reinterpret_cast<const uint16_t*>(Tk > 0 ? v : q);
  p.out = reinterpret_cast<uint16_t*>(out);
  p.q_st = q_st; p.q_sh = q_sh; p.k_st = k_st; p.k_sh = k_sh;
  p.v_st = v_st; p.v_sh = v_sh; p.o_st = o_st; p.o_sh = o_sh;
  p.Tq = Tq; p.Tk = Tk; p.Hq = Hq; p.Hkv = Hkv; p.G = Hq / Hkv; p.D = D;
  p.cu_q = cu_q; p.cu_k = cu_k; p.kv_lens = kv_lens;
  p.B = B;
  p.causal = causal != 0;
  p.zero_unowned = zero_unowned != 0;
  p.scale_log2 = scale * 1.4426950408889634f;
  cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_);
  const bool bf16 = dtype == OC_DT_BF16;
  const int dp = pl.dp, ctas = pl.ctas;
  if (pl.tile) {
    pl.tg.part = reinterpret_cast<float*>(workspace);
    if (dp == 64) return bf16 ? launch_tile<true, 64>(p, pl.tg, stream) : launch_tile<false, 64>(p, pl.tg, stream);
    if (dp == 128) return bf16 ? launch_tile<true, 128>(p, pl.tg, stream) : launch_tile<false, 128>(p, pl.tg, stream);
    return bf16 ? launch_tile<true, 256>(p, pl.tg, stream) : launch_tile<false, 256>(p, pl.tg, stream);
  }
  p.desc = reinterpret_cast<int*>(workspace);
  p.part = reinterpret_cast<float*>(reinterpret_cast<uint8_t*>(workspace) + split_desc_bytes(ctas));
  if (dp == 64) return bf16 ? launch_split<true, 64>(p, ctas, stream) : launch_split<false, 64>(p, ctas, stream);
  if (dp == 128) return bf16 ? launch_split<true, 128>(p, ctas, stream) : launch_split<false, 128>(p, ctas, stream);
  return bf16 ? launch_split<true, 256>(p, ctas, stream) : launch_split<false, 256>(p, ctas, stream);
}

extern "C" int oc_b200_dense_gemm_tile(int M, int N, int K, int* tokens, int* splits_k) {
  if (!tokens || !splits_k) return fail(OC_ERR_INVALID, "dense_gemm_tile: NULL pointer");
  if (M <= 0 || N <= 0 || K <= 0 || too_many(M) || too_many(N) || too_many(K))
    return fail(OC_ERR_INVALID, "dense_gemm_tile: M=%d N=%d K=%d (above 0, below 2^30)", M, N, K);
  int dev = 0;
  if (int rc = current_device(&dev)) return rc;
  *tokens = dense_split_tokens(M, N, K);
  *splits_k = *tokens != 0;
  if (!*tokens) *tokens = dense_bt(M, (N + 255) / 256, K, sm_count(dev) / 2);
  return OC_OK;
}

extern "C" int oc_b200_dense_gemm(const void* x, int64_t ldx, const void* w, int64_t ldw, int dtype, int M, int N,
                                  int K, const void* bias, int bias_dtype, const void* residual, int64_t ldr, int act,
                                  void* c, int64_t ldc, oc_stream_t stream_) {
  if (!dt16(dtype)) return fail(OC_ERR_INVALID, "dense_gemm: dtype %d (f16 or bf16)", dtype);
  if (M < 0 || N < 0 || K <= 0 || K % 8 != 0)
    return fail(OC_ERR_INVALID, "dense_gemm: M=%d N=%d K=%d (K a multiple of 8)", M, N, K);
  if (too_many(M) || too_many(N) || too_many(K))
    return fail(OC_ERR_INVALID, "dense_gemm: M=%d N=%d K=%d (below 2^30)", M, N, K);
  if (act < OC_ACT_NONE || act > OC_ACT_RELU) return fail(OC_ERR_INVALID, "dense_gemm: act %d", act);
  if (bias && !dtf(bias_dtype)) return fail(OC_ERR_INVALID, "dense_gemm: bias dtype %d", bias_dtype);
  if (M == 0 || N == 0) return OC_OK;
  if (!x || !w || !c) return fail(OC_ERR_INVALID, "dense_gemm: NULL pointer");
  if (!aligned(x, 16) || !aligned(w, 16) || ldx % 8 != 0 || ldw % 8 != 0 || ldx < K || ldw < K)
    return fail(OC_ERR_INVALID, "dense_gemm: X and W rows must be 16-byte aligned (ldx=%lld ldw=%lld)", (long long)ldx,
                (long long)ldw);
  if (ldc < N || (residual && ldr < N))
    return fail(OC_ERR_INVALID, "dense_gemm: ldc=%lld ldr=%lld for N=%d", (long long)ldc, (long long)ldr, N);
  int dev = 0;
  if (int rc = current_device(&dev)) return rc;
  oc::DenseParams p{};
  p.M = M;
  p.N = N;
  p.K = K;
  p.bias = bias;
  p.bias_dtype = bias_dtype;
  p.residual = reinterpret_cast<const uint16_t*>(residual);
  p.ldr = ldr;
  p.act = act;
  p.out = reinterpret_cast<uint16_t*>(c);
  p.ldc = ldc;
  p.vec = aligned(c, 16) && ldc % 8 == 0 && (!residual || (aligned(residual, 16) && ldr % 8 == 0));
  cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_);
  return dtype == OC_DT_BF16 ? launch_dense<true>(x, ldx, w, ldw, p, dev, stream)
                             : launch_dense<false>(x, ldx, w, ldw, p, dev, stream);
}
