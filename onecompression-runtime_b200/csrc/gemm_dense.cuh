// Dense 16-bit linear with its epilogue: C[M, N] = act(X[M, K] W[N, K]^T + bias) + residual,
// fp32 accumulation and epilogue, one rounding.
#pragma once

#include "common.cuh"

namespace oc {

// Epilogue activations of the dense linear (the first two are Act's). Each is evaluated so that its
// relative error stays near fp32's where the value is small: tanh-GELU as v / (1 + e^-2u) instead of
// a difference of numbers close to 1, GELU through the normal distribution function. The fast exponential
// and division are off by 2^-16 at most, and by less where results are not tiny: below half a step (2^-11, 2^-8).
enum DenseAct : int { kDenseNone = 0, kDenseGeluTanh = 1, kDenseGelu = 2, kDenseSilu = 3, kDenseRelu = 4 };

__device__ __forceinline__ float dense_act(float v, int act) {
  if (act == kDenseGeluTanh) {
    const float u = 0.7978845608028654f * fmaf(0.044715f * v, v * v, v);
    return __fdividef(v, 1.f + __expf(-2.f * u));
  }
  if (act == kDenseGelu) return v * normcdff(v);
  if (act == kDenseSilu) return silu_f32(v);
  if (act == kDenseRelu) return v < 0.f ? 0.f : v;
  return v;
}

struct DenseParams {
  int M, N, K;
  const void* bias;
  int bias_dtype;
  const uint16_t* residual;
  long long ldr;
  int act;
  uint16_t* out;
  long long ldc;
  int vec;          // 16-byte accesses to out and residual rows
  int n_tiles_m;    // token tiles (the grid is feature tiles x token tiles, times the cluster)
};

// Few tokens: bound by reading W once. A tile is 128 features (the MMA's M, weights straight from
// TMA as the A operand) x BN tokens (its N). A cluster of S CTAs splits K, so that few tiles still
// use every SM; the CTAs leave their fp32 accumulators in shared memory and each finishes BN / S
// tokens by adding the cluster's accumulators over distributed shared memory in rank order (no
// workspace, no atomics, the same bits on every run).
constexpr int kDsThreads = 192;   // warps 0-3: accumulator and epilogue, 4: TMA, 5: MMA

template <int BN> struct DsCfg {
  static constexpr int kWBytes = 128 * 128;                  // 128 features x 64 k
  static constexpr int kXBytes = BN * 128;
  static constexpr int kStageBytes = kWBytes + kXBytes;
  static constexpr int kAccBytes = BN * 128 * 4;
  static constexpr int kBudget = BN <= 64 ? 98304 : 196608;  // two CTAs per SM up to 64 tokens
  static constexpr int kStages = kBudget / kStageBytes;
  static constexpr int kRing = kStages * kStageBytes;
  static constexpr int kSmem = (kRing > kAccBytes ? kRing : kAccBytes) + 1024 + (2 * kStages + 1) * 8 + 16;
  static constexpr int kTmemCols = BN < 32 ? 32 : BN;
  static_assert(kSmem <= 232448, "shared memory per CTA");
};

template <bool BF16, int BN>
__global__ void __launch_bounds__(kDsThreads)
    dense_split_kernel(const __grid_constant__ CUtensorMap tmap_w, const __grid_constant__ CUtensorMap tmap_x,
                       const DenseParams p) {
  using Cfg = DsCfg<BN>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  constexpr int kDataBytes = Cfg::kRing > Cfg::kAccBytes ? Cfg::kRing : Cfg::kAccBytes;
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + kDataBytes);
  uint64_t* empty = full + Cfg::kStages;
  uint64_t* done = empty + Cfg::kStages;
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(done + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_holder + 1);
  const int warp = warp_uniform(warp_id()), lane = lane_id();
  uint32_t rank, S;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(S));
  const int tile = blockIdx.x / S;
  const int n0 = (tile / p.n_tiles_m) * 128, m0 = (tile % p.n_tiles_m) * BN;
  const int kb_all = (p.K + 63) / 64;
  const int kb0 = (int)((long long)kb_all * rank / S), kb1 = (int)((long long)kb_all * (rank + 1) / S);
  const int nkb = kb1 - kb0;

  if (threadIdx.x == 0) {
    for (int i = 0; i < Cfg::kStages; ++i) { mbar_init(&full[i], 1); mbar_init(&empty[i], 1); }
    mbar_init(done, 1);
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 5) {
    tmem_alloc(tmem_holder, Cfg::kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_holder;

  if (warp == 4) {
    const bool leader = elect_one();
    if (leader) {
      tma_prefetch_desc(&tmap_w);
      tma_prefetch_desc(&tmap_x);
    }
    int it = 0;
    for (int st = 0, par = 1; it < nkb; ++it) {
      if (!mbar_wait_warp(&empty[st], par, abort_flag, kDevErrTmaEmpty)) break;
      if (leader) {
        uint8_t* base = smem + st * Cfg::kStageBytes;
        mbar_arrive_expect_tx(&full[st], Cfg::kStageBytes);
        tma_load_2d(base, &tmap_w, &full[st], (kb0 + it) * 64, n0);
        tma_load_2d(base + Cfg::kWBytes, &tmap_x, &full[st], (kb0 + it) * 64, m0);
      }
      if (++st == Cfg::kStages) { st = 0; par ^= 1; }
    }
    // every load issued lands before the CTA goes on (consumed ones return at once)
    if (leader)
      for (int i = it > Cfg::kStages ? it - Cfg::kStages : 0; i < it; ++i)
        mbar_drain(&full[i % Cfg::kStages], (i / Cfg::kStages) & 1);
  } else if (warp == 5) {
    constexpr uint32_t idesc = make_idesc_f16(BF16, 128, BN);
    const uint32_t tm = warp_uniform(tmem);
    const uint64_t desc = smem_desc_kmajor_sw128(smem_u32(smem));   // counts in units of 16 bytes
    const bool leader = elect_one();
    for (int it = 0, st = 0, par = 0; it < nkb; ++it) {
      if (!mbar_wait_warp(&full[st], par, abort_flag, kDevErrTmaFull)) break;
      tc_fence_after();
      const uint64_t wd = desc + st * (Cfg::kStageBytes / 16), xd = wd + Cfg::kWBytes / 16;
      if (leader) {
#pragma unroll
        for (int j = 0; j < 4; ++j) tc_mma_ss(tm, wd + j * 2, xd + j * 2, idesc, (it | j) != 0 ? 1u : 0u);
        tc_commit(&empty[st]);
      }
      if (++st == Cfg::kStages) { st = 0; par ^= 1; }
    }
    if (leader) tc_commit(done);
  }
  __syncwarp();
  float* acc = reinterpret_cast<float*>(smem);   // [BN tokens][128 features]
  if (warp < 4) {
    mbar_wait(done, 0, abort_flag, kDevErrAccFull);
    tc_fence_after();
  }
  __syncthreads();   // the ring's loads and the MMAs that read it are done: the accumulator moves in
  if (warp < 4) {
    const int f = warp * 32 + lane;
#pragma unroll 1
    for (int c = 0; c < BN; c += 16) {
      uint32_t v[16];
      tmem_ld_32x32b_x16(tmem + ((uint32_t)(warp * 32) << 16) + (uint32_t)c, v);
      tc_wait_ld();
#pragma unroll
      for (int i = 0; i < 16; ++i) acc[(c + i) * 128 + f] = nkb > 0 ? __uint_as_float(v[i]) : 0.f;
    }
  }
  tc_fence_before();
  if (S > 1) cluster_sync_all(); else __syncthreads();
  if (warp == 5) {
    tc_fence_after();
    tmem_dealloc(tmem, Cfg::kTmemCols);
  }
  if (!*abort_flag) {
    // this CTA's tokens of the tile: 8 features of a token per thread
    const int per = (BN + (int)S - 1) / (int)S;
    const int t_begin = (int)rank * per, t_end = min(min(BN, t_begin + per), p.M - m0);
    uint32_t peer[8];
    for (uint32_t r = 0; r < S; ++r) peer[r & 7] = mapa_shared(acc, r);
    constexpr int kOdt = BF16 ? kBF16 : kF16;
    for (int i = threadIdx.x; i < (t_end - t_begin) * 16; i += kDsThreads) {
      const int t = t_begin + i / 16, f = (i % 16) * 8;
      const int n = n0 + f;
      if (n >= p.N) continue;
      float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
      if (S > 1) {
        for (uint32_t r = 0; r < S; ++r) {
          const float4 x = ld_dsmem_f4(peer[r & 7] + (t * 128 + f) * 4), y = ld_dsmem_f4(peer[r & 7] + (t * 128 + f) * 4 + 16);
          v[0] += x.x; v[1] += x.y; v[2] += x.z; v[3] += x.w;
          v[4] += y.x; v[5] += y.y; v[6] += y.z; v[7] += y.w;
        }
      } else {
        const float4 x = *reinterpret_cast<const float4*>(acc + t * 128 + f);
        const float4 y = *reinterpret_cast<const float4*>(acc + t * 128 + f + 4);
        v[0] = x.x; v[1] = x.y; v[2] = x.z; v[3] = x.w;
        v[4] = y.x; v[5] = y.y; v[6] = y.z; v[7] = y.w;
      }
      const long long m = m0 + t;
      uint16_t* dst = p.out + m * p.ldc + n;
      const uint16_t* res = p.residual ? p.residual + m * p.ldr + n : nullptr;
      const int nf = min(8, p.N - n);
      alignas(16) uint16_t rv[8];   // moved as one 16-byte vector where the rows allow
      if (res) {
        if (p.vec && nf == 8) {
          *reinterpret_cast<uint4*>(rv) = *reinterpret_cast<const uint4*>(res);
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (e < nf) rv[e] = res[e];
        }
      }
      alignas(16) uint16_t ov[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        if (e < nf) {
          float y = v[e] + (p.bias ? load_as_f32(p.bias, p.bias_dtype, n + e) : 0.f);
          y = dense_act(y, p.act);
          if (res) y += bits_to_f32(rv[e], kOdt);
          ov[e] = f32_to_bits(y, kOdt);
        }
      }
      if (p.vec && nf == 8) {
        *reinterpret_cast<uint4*>(dst) = *reinterpret_cast<const uint4*>(ov);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (e < nf) dst[e] = ov[e];
      }
    }
  }
  if (S > 1) cluster_sync_all();   // no CTA leaves while another reads its accumulator
}

// Many tokens: bound by the tensor pipe. Persistent pairs of CTAs (a cluster of two, one per SM) compute
// 256 features x up to 256 tokens with cta_group::2 MMAs: each CTA holds its 128 features' weights and
// half of the tokens' activations, so an SM moves 32 KB of shared memory per 128 x 256 x 64 product instead
// of 48 KB. Features are the MMA's M and tokens its N: a ragged token count is split into equal tiles
// of a multiple of 32 tokens. The accumulator is double
// buffered in TMEM, so four epilogue warps drain a tile while the next one is multiplied. Every epilogue
// warp owns 32 features (its TMEM lanes) and moves [32 tokens x 32 features] pieces through its own four
// buffers by TMA, residual pieces loaded two ahead; outputs or residuals that a tensor map cannot
// describe are stored directly.
constexpr int kDtThreads = 256;     // warp 0: TMA, 1: MMA, 4-7: epilogue
constexpr int kDtStages = 6;
constexpr int kDtBufs = 4;
constexpr int kDtPiece = 32 * 32 * 2;
constexpr int kDtStageBytes = 2 * 128 * 128;
constexpr int kDtBars = 2 * kDtStages + 2 * 2 + 1 + 4 * kDtBufs;
constexpr int kDtSmem = kDtStages * kDtStageBytes + 4 * kDtBufs * kDtPiece + 1024 + kDtBars * 8 + 16;
static_assert(kDtSmem <= 232448, "shared memory per CTA");

struct DenseTileParams {
  DenseParams d;
  int bt;                          // tokens of a tile, a multiple of 32 up to 256
  int tiles_n, tiles_m, tiles;     // 256-feature tiles, token tiles
  int tma_epi;
};

__device__ __forceinline__ void tc_mma_ss_pair(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                               uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}

// Tile number -> (feature tile, token tile): bands of 8 feature tiles, so that the pairs running at one
// time share both weights and activations in L2.
__device__ __forceinline__ void dense_tile_at(const DenseTileParams& p, int tile, int& tn, int& tm) {
  const int band = tile / (8 * p.tiles_m), in = tile - band * 8 * p.tiles_m;
  const int width = min(8, p.tiles_n - band * 8);
  tm = in / width;
  tn = band * 8 + in - tm * width;
}

template <bool BF16, int ACT, bool RES>
__device__ __forceinline__ void dense_piece(const uint32_t (&v)[32], float bias, uint16_t* e) {
  constexpr int kOdt = BF16 ? kBF16 : kF16;
#pragma unroll
  for (int i = 0; i < 32; ++i) {
    float y = dense_act(__uint_as_float(v[i]) + bias, ACT);
    if constexpr (RES) y += bits_to_f32(e[i * 32], kOdt);
    e[i * 32] = f32_to_bits(y, kOdt);
  }
}

template <bool BF16, int ACT, bool RES>
__global__ void __launch_bounds__(kDtThreads, 1)
    dense_tile_kernel(const __grid_constant__ CUtensorMap tmap_w, const __grid_constant__ CUtensorMap tmap_x,
                      const __grid_constant__ CUtensorMap tmap_c, const __grid_constant__ CUtensorMap tmap_r,
                      const DenseTileParams p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* epi = smem + kDtStages * kDtStageBytes;
  uint64_t* full = reinterpret_cast<uint64_t*>(epi + 4 * kDtBufs * kDtPiece);   // the leader's count both CTAs' loads
  uint64_t* empty = full + kDtStages;
  uint64_t* acc_full = empty + kDtStages;    // [2]
  uint64_t* acc_empty = acc_full + 2;        // [2] the leader's: one arrival per epilogue warp of both CTAs
  uint64_t* drain = acc_empty + 2;
  uint64_t* res_full = drain + 1;            // [4 warps][kDtBufs]
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(res_full + 4 * kDtBufs);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_holder + 1);
  const int warp = warp_uniform(warp_id()), lane = lane_id();
  const uint32_t rank = cluster_ctarank();
  const bool leader = rank == 0;
  const int tile0 = blockIdx.x / 2, step = gridDim.x / 2;
  const int KB = (p.d.K + 63) / 64;
  const int half = p.bt / 2;
  const uint32_t x_bytes = half * 128;

  if (threadIdx.x == 0) {
    for (int i = 0; i < kDtStages; ++i) { mbar_init(&full[i], 1); mbar_init(&empty[i], 1); }
    for (int i = 0; i < 2; ++i) { mbar_init(&acc_full[i], 1); mbar_init(&acc_empty[i], 8); }
    mbar_init(drain, 1);
    for (int i = 0; i < 4 * kDtBufs; ++i) mbar_init(&res_full[i], 1);
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 0 && lane == 0) {
    tma_prefetch_desc(&tmap_w);
    tma_prefetch_desc(&tmap_x);
    if (p.tma_epi) tma_prefetch_desc(&tmap_c);
    if (RES && p.tma_epi) tma_prefetch_desc(&tmap_r);
  }
  if (warp == 1) {
    tmem_alloc_cg2(tmem_holder, 512);
    tmem_relinquish_cg2();
  }
  tc_fence_before();
  cluster_sync_all();   // both CTAs' barriers are there before a copy or an arrival crosses over
  tc_fence_after();
  const uint32_t tmem = *tmem_holder;

  if (warp == 0) {
    const bool issue = elect_one();
    const uint32_t full0 = mapa_shared(full, 0);   // the leader's barriers
    const uint32_t tx = 2 * (128 * 128 + x_bytes);
    int it = 0;
    bool ok = true;
    for (int tile = tile0, st = 0, par = 1; ok && tile < p.tiles; tile += step) {
      int tn, tm;
      dense_tile_at(p, tile, tn, tm);
      const int f0 = tn * 256 + (int)rank * 128, t0 = tm * p.bt + (int)rank * half;
      for (int kb = 0; kb < KB; ++kb, ++it) {
        if (!mbar_wait_warp(&empty[st], par, abort_flag, kDevErrTmaEmpty)) { ok = false; break; }
        if (issue) {
          if (leader) mbar_arrive_expect_tx(&full[st], tx);
          uint8_t* base = smem + st * kDtStageBytes;
          tma_load_2d_pair(base, &tmap_w, full0 + st * 8, kb * 64, f0);
          tma_load_2d_pair(base + 128 * 128, &tmap_x, full0 + st * 8, kb * 64, t0);
        }
        if (++st == kDtStages) { st = 0; par ^= 1; }
      }
    }
    // our copies signal the leader's barrier: wait until the pair's MMAs have released the stages
    // we filled, then every copy has landed
    if (issue)
      for (int i = it > kDtStages ? it - kDtStages : 0; i < it; ++i)
        mbar_drain(&empty[i % kDtStages], (i / kDtStages) & 1);
  } else if (warp == 1) {
    if (leader) {   // the whole warp runs with uniform values, one elected thread issues
      const uint32_t idesc = make_idesc_f16(BF16, 256, p.bt);
      const uint32_t tb = warp_uniform(tmem);
      const uint64_t desc = smem_desc_kmajor_sw128(smem_u32(smem));   // counts in units of 16 bytes
      const bool issue = elect_one();
      int n = 0;
      bool ok = true;
      for (int tile = tile0, st = 0, par = 0; ok && tile < p.tiles; tile += step, ++n) {
        const int a = n & 1;
        if (!__all_sync(0xffffffffu, mbar_wait_cluster_ns(&acc_empty[a], ((n >> 1) & 1) ^ 1, kDevErrAccEmpty, OC_WAIT_NS))) {
          *abort_flag = 1;
          break;
        }
        tc_fence_after();
        for (int kb = 0; kb < KB; ++kb) {
          if (!mbar_wait_warp(&full[st], par, abort_flag, kDevErrTmaFull)) { ok = false; break; }
          tc_fence_after();
          const uint64_t wd = desc + st * (kDtStageBytes / 16), xd = wd + 128 * 128 / 16;
          if (issue) {
#pragma unroll
            for (int j = 0; j < 4; ++j)
              tc_mma_ss_pair(tb + a * 256, wd + j * 2, xd + j * 2, idesc, (kb | j) != 0 ? 1u : 0u);
            tc_commit_pair(&empty[st], 0x3);
          }
          if (++st == kDtStages) { st = 0; par ^= 1; }
        }
        if (ok && issue) tc_commit_pair(&acc_full[a], 0x3);
      }
      if (issue) {
        tc_commit_pair(drain, 0x1);
        mbar_drain(drain, 0);
      }
      __syncwarp();
    }
  } else if (warp >= 4) {
    const int q4 = warp & 3;
    uint16_t* bufs = reinterpret_cast<uint16_t*>(epi) + q4 * (kDtBufs * kDtPiece / 2);
    uint64_t* rbar = res_full + q4 * kDtBufs;
    uint32_t piece = 0;              // running piece counter: buffer piece & 3
    uint32_t pend = 0, pend_par = 0; // lane 0: residual loads in flight, their phases
    int n = 0;
    auto load_res = [&](uint32_t pc, int f0, int t0) {
      const int b = pc & (kDtBufs - 1);
      mbar_arrive_expect_tx(&rbar[b], kDtPiece);
      tma_load_2d(bufs + b * (kDtPiece / 2), &tmap_r, &rbar[b], f0, t0);
      pend |= 1u << b;
      pend_par = (pend_par & ~(1u << b)) | (((pc / kDtBufs) & 1u) << b);
    };
    for (int tile = tile0; tile < p.tiles; tile += step, ++n) {
      int tn, tm;
      dense_tile_at(p, tile, tn, tm);
      const int a = n & 1;
      const int f0 = tn * 256 + (int)rank * 128 + q4 * 32, t0 = tm * p.bt;
      const int f = f0 + lane;
      const float bias = p.d.bias && f < p.d.N ? load_as_f32(p.d.bias, p.d.bias_dtype, f) : 0.f;
      // pieces that hold anything: the ragged last tiles stop early
      const int pieces = f0 < p.d.N ? (min(p.bt, p.d.M - t0) + 31) / 32 : 0;
      if (p.tma_epi && lane == 0) {
        bulk_wait_group_read<2>();   // the stores of pieces piece - 4 and - 3 have read their buffers
        if (RES)
          for (int c = 0; c < 2 && c < pieces; ++c) load_res(piece + c, f0, t0 + c * 32);
      }
      __syncwarp();
      bool ok = __all_sync(0xffffffffu, mbar_wait(&acc_full[a], (n >> 1) & 1, abort_flag, kDevErrAccFull));
      if (!ok) break;
      tc_fence_after();
      const uint32_t acc = tmem + ((uint32_t)(q4 * 32) << 16) + (uint32_t)(a * 256);
#pragma unroll 1
      for (int c = 0; c < pieces; ++c) {
        uint32_t v[32];
        tmem_ld_32x32b_x32(acc + (uint32_t)(c * 32), v);
        if (p.tma_epi) {
          const int b = piece & (kDtBufs - 1);
          if (lane == 0 && c + 2 < pieces) {
            bulk_wait_group_read<1>();   // the store of piece - 2 has read the buffer of piece + 2
            if (RES) load_res(piece + 2, f0, t0 + (c + 2) * 32);
          }
          tc_wait_ld();
          if constexpr (RES) {
            ok = __all_sync(0xffffffffu, mbar_wait(&rbar[b], (piece / kDtBufs) & 1, abort_flag, kDevErrResFull));
            if (!ok) break;
            if (lane == 0) pend &= ~(1u << b);
          }
          __syncwarp();
          dense_piece<BF16, ACT, RES>(v, bias, bufs + b * (kDtPiece / 2) + lane);
          fence_proxy_async_shared();
          __syncwarp();
          if (lane == 0) {
            tma_store_2d(&tmap_c, bufs + b * (kDtPiece / 2), f0, t0 + c * 32);
            bulk_commit_group();
          }
          ++piece;
        } else {
          tc_wait_ld();
          constexpr int kOdt = BF16 ? kBF16 : kF16;
          if (f < p.d.N) {
            const int rows = min(32, p.d.M - t0 - c * 32);
            uint16_t* dst = p.d.out + (long long)(t0 + c * 32) * p.d.ldc + f;
            const uint16_t* res = RES ? p.d.residual + (long long)(t0 + c * 32) * p.d.ldr + f : nullptr;
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (i < rows) {
                float y = dense_act(__uint_as_float(v[i]) + bias, ACT);
                if constexpr (RES) y += bits_to_f32(res[i * p.d.ldr], kOdt);
                dst[i * p.d.ldc] = f32_to_bits(y, kOdt);
              }
          }
        }
      }
      if (!ok) break;
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_cluster(mapa_shared(&acc_empty[a], 0));
    }
    if (lane == 0) {
      bulk_wait_group0();
      for (int b = 0; b < kDtBufs; ++b)
        if (pend & (1u << b)) mbar_drain(&rbar[b], (pend_par >> b) & 1u);
    }
  }

  tc_fence_before();
  cluster_sync_all();   // neither CTA leaves, or frees TMEM, while the pair's MMAs or arrivals may touch it
  if (warp == 1) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc_cg2(tmem, 512);
  }
}

}  // namespace oc
