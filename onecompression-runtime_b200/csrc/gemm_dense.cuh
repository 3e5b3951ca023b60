// Dense 16-bit linear with its epilogue: C[M, N] = act(X[M, K] W[N, K]^T + bias) + residual,
// fp32 accumulation and epilogue, one rounding.
#pragma once

#include "common.cuh"

namespace oc {

// Epilogue activations of the dense linear (the first two are Act's). Each is evaluated so that its
// relative error stays near fp32's where the value is small: tanh-GELU as v / (1 + e^-2u) instead of
// a difference of numbers close to 1, GELU through the normal distribution function.
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
  const int warp = warp_id(), lane = lane_id();
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
    if (lane == 0) {
      tma_prefetch_desc(&tmap_w);
      tma_prefetch_desc(&tmap_x);
      int it = 0;
      for (; it < nkb; ++it) {
        const int st = it % Cfg::kStages;
        if (!mbar_wait(&empty[st], ((it / Cfg::kStages) & 1) ^ 1, abort_flag, kDevErrTmaEmpty)) break;
        uint8_t* base = smem + st * Cfg::kStageBytes;
        mbar_arrive_expect_tx(&full[st], Cfg::kStageBytes);
        tma_load_2d(base, &tmap_w, &full[st], (kb0 + it) * 64, n0);
        tma_load_2d(base + Cfg::kWBytes, &tmap_x, &full[st], (kb0 + it) * 64, m0);
      }
      // every load issued lands before the CTA goes on (consumed ones return at once)
      for (int i = it > Cfg::kStages ? it - Cfg::kStages : 0; i < it; ++i)
        mbar_drain(&full[i % Cfg::kStages], (i / Cfg::kStages) & 1);
    }
  } else if (warp == 5) {
    if (lane == 0) {
      constexpr uint32_t idesc = make_idesc_f16(BF16, 128, BN);
      for (int it = 0; it < nkb; ++it) {
        const int st = it % Cfg::kStages;
        if (!mbar_wait(&full[st], (it / Cfg::kStages) & 1, abort_flag, kDevErrTmaFull)) break;
        tc_fence_after();
        const uint32_t wa = smem_u32(smem + st * Cfg::kStageBytes), xa = wa + Cfg::kWBytes;
#pragma unroll
        for (int j = 0; j < 4; ++j)
          tc_mma_ss(tmem, smem_desc_kmajor_sw128(wa + j * 32), smem_desc_kmajor_sw128(xa + j * 32), idesc,
                    (it | j) != 0 ? 1u : 0u);
        tc_commit(&empty[st]);
      }
      tc_commit(done);
    }
  }
  __syncwarp();
  bool ok = true;
  float* acc = reinterpret_cast<float*>(smem);   // [BN tokens][128 features]
  if (warp < 4) {
    ok = mbar_wait(done, 0, abort_flag, kDevErrAccFull);
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
      uint16_t rv[8];
      if (res) {
        if (p.vec && nf == 8) {
          *reinterpret_cast<uint4*>(rv) = *reinterpret_cast<const uint4*>(res);
        } else {
          for (int e = 0; e < nf; ++e) rv[e] = res[e];
        }
      }
      uint16_t ov[8];
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
        for (int e = 0; e < nf; ++e) dst[e] = ov[e];
      }
    }
  }
  if (S > 1) cluster_sync_all();   // no CTA leaves while another reads its accumulator
}

}  // namespace oc
