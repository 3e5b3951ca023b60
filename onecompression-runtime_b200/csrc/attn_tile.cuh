// Attention for prompts: many query rows per sequence, on the 5th-generation tensor cores.
//
// Bound by the tensor pipe and, at head size 64 and 128, by the exponentials (16 a cycle and SM against
// 8192 tensor operations). The (token, head) rows of a key head's query heads are packed into tiles of
// 128 rows, two tiles to a CTA (one where the head size is 256): S = Q K^T and O += P V as tcgen05 MMAs of
// 128 x 128 x 16 into TMEM, one pass over the keys in blocks of 128.
//   * A softmax warpgroup per tile, one thread per row: it reads S from TMEM (no shuffles), writes the
//     weights P back to TMEM as the A operand of the second product, and keeps maximum and sum in registers.
//     P is rounded to 16 bits once, as the product takes it (half a step of each weight; the sum adds
//     the unrounded ones, so the error does not grow with the keys).
//   * One warp issues both tiles' products in turn: while one tile is in its softmax the tensor pipe runs
//     the other's, and the second product starts on the first 96 keys' weights while the softmax works
//     on the rest.
//   * The reference that the exponents are taken against follows the running maximum only when
//     it grows by more than 2^8: weights up to 256 are as exact in 16 bits as weights up to 1, and
//     the accumulator in TMEM is read, scaled and written back only in those rare steps.
//   * K and V move by TMA in units of [128 keys x 64 columns] (128-byte swizzle) through one ring that
//     both tiles of the CTA share; V is read by the MMA in its own layout (MN-major B operand).
//   * Two warps prepare the V blocks at the end of what the rows see (the causal diagonal, the end
//     of the sequence): rows behind the keys become zeros, and in causal blocks infinities and NaN,
//     which a weight of zero must not turn into NaN, are taken out and added afterwards by the rows
//     that see them.
// Tiles are numbered without the host knowing a length: sequence b's CTAs start at
// floor(cu_q[b] / tokens) + b, which leaves room for every sequence's ragged last tile; a CTA whose tokens
// lie behind its sequence's end exits. Every head's tiles run from its last token up, so that the long
// causal tiles start first. Where the tiles of a call would leave SMs idle, several CTAs take a part of
// the keys each and leave fp32 partials that attn_tile_join_kernel adds in order. All waits are bounded
// (common.cuh).
#pragma once

#include "attn_common.cuh"

namespace oc {

constexpr int kTileKeys = 128;
constexpr int kTileUnitBytes = 128 * 128;   // [128 rows x 64 columns] of 16-bit values
constexpr int kTileMaxEdges = 3;
constexpr int kTileNegate = 1, kTileZeroScale = 2;   // of a negative and a zero softmax scale
template <int DP> struct TileCfg {
  static constexpr int kTiles = DP == 256 ? 1 : 2;          // row tiles of a CTA
  static constexpr int kRows = kTiles * 128;
  static constexpr int kUnits = DP / 64;                    // units of a K or V block
  static constexpr int kSlots = DP == 256 ? 2 : DP == 128 ? 5 : 10;
  static constexpr int kGroup = DP == 256 ? 1 : kUnits;     // units that share a barrier: few blocks fit at 256,
                                                            // where loads follow the products unit by unit
  static constexpr int kGroups = kUnits / kGroup;
  static constexpr int kSoftmaxThreads = kTiles * 128;
  static constexpr int kSoftmaxRegs = 216, kAuxRegs = 72;   // of two tiles: 168 at launch for each of 384 threads
  static constexpr int kThreads = kSoftmaxThreads + 128;
  static constexpr int kQBytes = kTiles * kUnits * kTileUnitBytes;
  static constexpr int kRingBytes = kSlots * kUnits * kTileUnitBytes;
  static constexpr int kBars = 2 * kSlots * kGroups + 1 + 2 + 2 + 2 + 2 + 2 * kTileMaxEdges + 1;
  static constexpr int kSmem = kQBytes + kRingBytes + 1024 + kBars * 8 + 32;
  static constexpr uint32_t kOCol = 256;
  __device__ static constexpr uint32_t s_col(int i) { return i * 128; }
  // P shares the columns of its S (read by then), except where the head leaves TMEM to spare
  __device__ static constexpr uint32_t p_col(int i) { return DP == 64 ? 384 + i * 64 : i * 128; }
  __device__ static constexpr uint32_t o_col(int t) { return kOCol + t * DP; }
  static_assert(kSmem <= 232448, "shared memory per CTA");
};

__device__ __forceinline__ void tma_load_3d(void* dst, const CUtensorMap* map, uint64_t* bar, int x, int y, int z) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(
          smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(x), "r"(y), "r"(z)
      : "memory");
}

// MN-major operand with the 128-byte swizzle: rows of 64 values along N (128 B), 8-row atoms along K
// 1024 B apart, groups of 64 along N one unit apart.
__device__ __forceinline__ uint64_t smem_desc_mnmajor_sw128(uint32_t addr) {
  uint64_t d = 0;
  d |= (uint64_t)((addr & 0x3FFFFu) >> 4);
  d |= (uint64_t)(kTileUnitBytes >> 4) << 16;
  d |= (uint64_t)(1024u >> 4) << 32;
  d |= (uint64_t)1 << 46;
  d |= (uint64_t)2 << 61;
  return d;
}

__device__ __forceinline__ void tmem_st_32x32b_x16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}

struct TileMaps { CUtensorMap q, k, v; };

struct TileGrid {
  int tokens;    // of a tile: 128 / G
  int slots;     // CTAs' token ranges over all sequences, ragged ends included
  int splits;    // CTAs that share the keys of a range
  float* part;   // splits > 1: [key head, slot][split][tile], each O [DP][128 rows], m [128], l [128]: a warp's rows
                 // lie side by side (row by row, 8-byte stores 520 B apart doubled the time of a split prompt)
};

// What a CTA works on; every role derives the same numbers. With a split, the keys are those of its part:
// the sequence's key rows then start at the part's first block.
struct TileWork {
  Seq s;
  int kvh, t0, ntile, nblk, e0, split;   // t0: first token; e0: first block that some row does not see whole
  int nb[2];                             // blocks of each tile
};

// The sequence and first token of a token range; false behind the sequence's end. A whole warp searches: its
// lanes look at 32 places of the table at a time, one load's latency for up to 32 sequences.
template <int DP> __device__ __forceinline__ bool tile_range(const AttnParams& p, const TileGrid& tg, int slot, TileWork& w) {
  const int R = TileCfg<DP>::kTiles * tg.tokens;
  int lo = 0, n = p.B;   // the last sequence of [lo, lo + n) that starts at or before the slot
  while (n > 1) {
    const int step = (n + 31) / 32, at = lane_id() * step;
    const bool before = at < n && (p.cu_q ? min(max(p.cu_q[lo + at], 0), p.Tq) : 0) / R + lo + at <= slot;
    const unsigned mask = __ballot_sync(0xffffffffu, before);
    const int k = mask ? 31 - __clz(mask) : 0;
    lo += k * step;
    n = min(step, n - k * step);
  }
  w.s = attn_seq(p, lo);
  const long long t0 = (long long)(slot - (w.s.q0 / R + lo)) * R;
  if (t0 < 0 || t0 >= w.s.nq) return false;
  w.t0 = (int)t0;
  w.ntile = min(TileCfg<DP>::kTiles, (w.s.nq - w.t0 + tg.tokens - 1) / tg.tokens);
  return true;
}

template <int DP> __device__ __forceinline__ bool tile_work(const AttnParams& p, const TileGrid& tg, TileWork& w) {
  const int unit = blockIdx.x / tg.splits;
  w.split = blockIdx.x - unit * tg.splits;
  w.kvh = unit / tg.slots;
  if (!tile_range<DP>(p, tg, tg.slots - 1 - (unit - w.kvh * tg.slots), w)) return false;
  const int off = w.s.nk - w.s.nq;
  auto blocks = [&](int t) {   // that the tile's last token sees
    const int last = min(w.s.nq, w.t0 + (t + 1) * tg.tokens) - 1;
    const int keys = p.causal ? min(w.s.nk, max(0, last + off + 1)) : w.s.nk;
    return (keys + kTileKeys - 1) / kTileKeys;
  };
  const int all = blocks(w.ntile - 1);
  const int j0 = (int)((long long)all * w.split / tg.splits), j1 = (int)((long long)all * (w.split + 1) / tg.splits);
  for (int t = 0; t < 2; ++t) w.nb[t] = t < w.ntile ? max(0, min(blocks(t), j1) - j0) : 0;
  w.nblk = w.nb[w.ntile - 1];
  const int whole = (p.causal ? max(0, min(w.s.nk, w.t0 + off + 1)) : w.s.nk) / kTileKeys;   // blocks the first row sees
  w.e0 = min(max(whole - j0, 0), w.nblk);
  w.s.k0 += j0 * kTileKeys;
  w.s.nk -= j0 * kTileKeys;
  return true;
}

// Sequence number in the ring of block j's K and V loads, in the order the MMAs take them.
template <int DP> __device__ __forceinline__ int k_use(int j) { return TileCfg<DP>::kTiles == 2 || j == 0 ? 2 * j : 2 * j - 1; }
template <int DP> __device__ __forceinline__ int v_use(int j, int nblk) {
  return TileCfg<DP>::kTiles == 2 || j == nblk - 1 ? 2 * j + 1 : 2 * j + 2;
}

template <bool BF16, int DP>
__global__ void __launch_bounds__(TileCfg<DP>::kThreads, 1)
    attn_tile_kernel(const __grid_constant__ TileMaps maps, const AttnParams p, const TileGrid tg, const int mode) {
  using Cfg = TileCfg<DP>;
  constexpr int U = Cfg::kUnits, GU = Cfg::kGroup, GN = Cfg::kGroups, NB = Cfg::kSlots * GN;
  constexpr bool kTwo = Cfg::kTiles == 2;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* q_smem = smem;
  uint8_t* ring = smem + Cfg::kQBytes;
  uint64_t* full = reinterpret_cast<uint64_t*>(ring + Cfg::kRingBytes);
  uint64_t* empty = full + NB;
  uint64_t* q_full = empty + NB;
  uint64_t* s_full = q_full + 1;            // [2] by tile, or by block parity where there is one tile
  uint64_t* p_part = s_full + 2;            // [2] the first 96 keys' weights are there
  uint64_t* p_full = p_part + 2;            // [2] all are
  uint64_t* pv_done = p_full + 2;           // [2] by tile
  uint64_t* edge_full = pv_done + 2;        // [3] V blocks from e0 on: loaded
  uint64_t* edge_ready = edge_full + kTileMaxEdges;   // [3] and prepared
  uint64_t* drain = edge_ready + kTileMaxEdges;
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(drain + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_holder + 1);
  volatile int* odd_values = abort_flag + 1;   // an infinity or NaN was taken out of a V block
  const int warp = warp_uniform(warp_id()), lane = lane_id();

  TileWork w;
  const bool work = tile_work<DP>(p, tg, w);
  if (blockIdx.x == 0)
    for (int b = threadIdx.x; b < p.B; b += Cfg::kThreads) attn_seq(p, b, true);
  if (!work) {
    const bool none = __syncthreads_or(attn_disorder(p, threadIdx.x, Cfg::kThreads));
    if (p.zero_unowned) attn_zero_unowned(p, none, blockIdx.x, gridDim.x, threadIdx.x, Cfg::kThreads);
    return;
  }
  const Seq s = w.s;
  const int off = s.nk - s.nq;   // the same for a part of the keys, counted from its first

  if (threadIdx.x == 0) {
    for (int i = 0; i < NB; ++i) { mbar_init(&full[i], 1); mbar_init(&empty[i], 1); }
    mbar_init(q_full, 1);
    for (int i = 0; i < 2; ++i) { mbar_init(&s_full[i], 1); mbar_init(&p_part[i], 128); mbar_init(&p_full[i], 128); mbar_init(&pv_done[i], 1); }
    for (int i = 0; i < kTileMaxEdges; ++i) { mbar_init(&edge_full[i], 1); mbar_init(&edge_ready[i], 64); }
    mbar_init(drain, 1);
    *abort_flag = 0;
    *odd_values = 0;
    fence_barrier_init();
  }
  constexpr int kAux = Cfg::kSoftmaxThreads / 32;   // first warp of the last warpgroup: TMA, MMA, V, V
  if (warp == kAux + 1) {
    tmem_alloc(tmem_holder, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  const bool none = __syncthreads_or(attn_disorder(p, threadIdx.x, Cfg::kThreads));
  tc_fence_after();
  const uint32_t tmem = *tmem_holder;
  if (none) {   // the table decreases: nothing is run
    if (p.zero_unowned) attn_zero_unowned(p, true, blockIdx.x, gridDim.x, threadIdx.x, Cfg::kThreads);
    if (tg.splits > 1 && threadIdx.x < Cfg::kRows)   // a sum of weights that no row has: the join leaves such rows alone
      tg.part[((long long)blockIdx.x * Cfg::kTiles + threadIdx.x / 128) * (128 * (DP + 2)) + (DP + 1) * 128 +
              threadIdx.x % 128] = -1.f;
    if (warp == kAux + 1) tmem_dealloc(tmem, 512);
    return;
  }

  if (warp >= kAux) {
    if constexpr (kTwo) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(Cfg::kAuxRegs));
    if (warp == kAux) {
      // ------------------------------------------------------------ TMA
      if (lane == 0) {
        tma_prefetch_desc(&maps.q);
        tma_prefetch_desc(&maps.k);
        tma_prefetch_desc(&maps.v);
        mbar_arrive_expect_tx(q_full, w.ntile * U * tg.tokens * p.G * 128);
        for (int t = 0; t < w.ntile; ++t)
          for (int u = 0; u < U; ++u)   // row token * G + head of the tile
            tma_load_3d(q_smem + (t * U + u) * kTileUnitBytes, &maps.q, q_full, u * 64, w.kvh * p.G,
                        s.q0 + w.t0 + t * tg.tokens);
        int edges = 0, uses = 0;
        bool ok = true;
        for (int n = 0; ok && n < 2 * w.nblk; ++n) {
          // the n-th block in the MMAs' order
          int j = n >> 1;
          bool is_v = n & 1;
          if (!kTwo && n > 0 && n < 2 * w.nblk - 1) { is_v = !(n & 1); j = is_v ? (n - 2) >> 1 : (n + 1) >> 1; }
          const int slot = n % Cfg::kSlots, par = (n / Cfg::kSlots) & 1;
          const bool edge = is_v && j >= w.e0;
          if (edge) {
            mbar_arrive_expect_tx(&edge_full[j - w.e0], U * kTileUnitBytes);
            ++edges;
          }
          for (int g = 0; g < GN; ++g) {
            const int i = slot * GN + g;
            if (!mbar_wait(&empty[i], par ^ 1, abort_flag, kDevErrTmaEmpty)) {
              // an edge block was announced: its remaining bytes never come, so nobody drains it
              if (edge) --edges;
              ok = false;
              break;
            }
            uint64_t* bar = edge ? &edge_full[j - w.e0] : &full[i];
            if (edge) mbar_arrive(&full[i]);   // the ring's phases go on; the block is announced on its own barrier
            else mbar_arrive_expect_tx(&full[i], GU * kTileUnitBytes);
            for (int u = g * GU; u < (g + 1) * GU; ++u)
              tma_load_3d(ring + (slot * U + u) * kTileUnitBytes, is_v ? &maps.v : &maps.k, bar, u * 64, w.kvh,
                          s.k0 + j * kTileKeys);
            ++uses;
          }
        }
        // every load issued lands before the CTA exits (consumed ones return at once)
        mbar_drain(q_full, 0);
        for (int i = uses > NB ? uses - NB : 0; i < uses; ++i) mbar_drain(&full[i % NB], (i / NB) & 1);
        for (int e = 0; e < edges; ++e) mbar_drain(&edge_full[e], 0);
      }
    } else if (warp == kAux + 1) {
      // ------------------------------------------------------------ MMA
      // The whole warp runs this with warp-uniform values; one elected thread issues.
      const uint32_t idesc_qk = make_idesc_f16(BF16, 128, 128) | (mode & kTileNegate ? 1u << 13 : 0u);
      constexpr uint32_t idesc_pv = make_idesc_f16(BF16, 128, DP) | (1u << 16);   // B is MN-major
      const int last_tile = warp_uniform(w.ntile - 1), nblk = warp_uniform(w.nblk), e0 = warp_uniform(w.e0);
      const int nb0 = warp_uniform(w.nb[0]);
      const uint32_t tm = warp_uniform(tmem);
      const uint64_t q_desc = smem_desc_kmajor_sw128(smem_u32(q_smem));
      const uint64_t k_desc = smem_desc_kmajor_sw128(smem_u32(ring)), v_desc = smem_desc_mnmajor_sw128(smem_u32(ring));
      // `first`: no other tile has waited for the block yet
      auto qk = [&](const int t, const int j, const bool first) {
        const int n = k_use<DP>(j), slot = n % Cfg::kSlots, par = (n / Cfg::kSlots) & 1;
        const int b = kTwo ? t : (j & 1);
#pragma unroll
        for (int g = 0; g < GN; ++g) {
          if (first && !mbar_wait_warp(&full[slot * GN + g], par, abort_flag, kDevErrTmaFull)) return false;
          tc_fence_after();
          if (elect_one()) {
#pragma unroll
            for (int u = g * GU; u < (g + 1) * GU; ++u)
#pragma unroll
              for (int k = 0; k < 4; ++k)   // descriptors count in units of 16 bytes
                tc_mma_ss(tm + Cfg::s_col(b), q_desc + (t * U + u) * (kTileUnitBytes / 16) + k * 2,
                          k_desc + (slot * U + u) * (kTileUnitBytes / 16) + k * 2, idesc_qk, (u | k) != 0 ? 1u : 0u);
            if (g == GN - 1) tc_commit(&s_full[b]);
            if (t == last_tile) tc_commit(&empty[slot * GN + g]);
          }
          __syncwarp();
        }
        return true;
      };
      auto pv = [&](const int t, const int j, const bool first) {
        const int n = v_use<DP>(j, nblk), slot = n % Cfg::kSlots, par = (n / Cfg::kSlots) & 1;
        const int b = kTwo ? t : (j & 1);
        const uint32_t pp = kTwo ? (j & 1) : ((j >> 1) & 1);
        if (first) {
          if (j >= e0) {
            if (!mbar_wait_warp(&edge_ready[j - e0], 0, abort_flag, kDevErrWFull)) return false;
          } else {
#pragma unroll
            for (int g = 0; g < GN; ++g)
              if (!mbar_wait_warp(&full[slot * GN + g], par, abort_flag, kDevErrTmaFull)) return false;
          }
        }
        const uint64_t vd = v_desc + slot * U * (kTileUnitBytes / 16);
#pragma unroll
        for (int h = 0; h < 2; ++h) {   // the first keys' weights while the softmax still works on the others
          if (!mbar_wait_warp(h ? &p_full[b] : &p_part[b], pp, abort_flag, kDevErrAFull)) return false;
          tc_fence_after();
          if (elect_one()) {
#pragma unroll
            for (int k = h ? 6 : 0; k < (h ? 8 : 6); ++k)
              tc_mma_ts(tm + Cfg::o_col(t), tm + Cfg::p_col(b) + k * 8, vd + k * (2048 / 16), idesc_pv,
                        (j | k) != 0 ? 1u : 0u);
            if (h) {
              tc_commit(&pv_done[t]);
              if (t == last_tile)
#pragma unroll
                for (int g = 0; g < GN; ++g) tc_commit(&empty[slot * GN + g]);
            }
          }
          __syncwarp();
        }
        return true;
      };
      // S(j + 1) overwrites the columns of P(j) (two tiles) or P(j - 1) (one tile): only once the
      // product that reads them is done. Where P has columns of its own (head size 64) the product before
      // is waited for instead. A wait by parity tells a phase from the one before it only, so every wait on
      // pv_done needs the knowledge that the phase before is over and that the one behind it cannot be:
      // this warp sees phase j - 1 before it issues PV(j), and S(j + 1), issued later, carries that to the softmax.
      auto pv_over = [&](const int t, const int j) {
        return mbar_wait_warp(&pv_done[t], j & 1, abort_flag, kDevErrAccFull);
      };
      bool ok = mbar_wait_warp(q_full, 0, abort_flag, kDevErrResFull);
      if constexpr (kTwo) {
        if (ok && nb0 > 0) ok = qk(0, 0, true);
        if (ok && last_tile && nblk > 0) ok = qk(1, 0, nb0 == 0);
        for (int j = 0; ok && j < nblk; ++j) {
          if (j < nb0) ok = (DP != 64 || j == 0 || pv_over(0, j - 1)) && pv(0, j, true);
          if (ok && j + 1 < nb0) ok = (DP == 64 || pv_over(0, j)) && qk(0, j + 1, true);
          if (!last_tile) continue;
          if (ok) ok = (DP != 64 || j == 0 || pv_over(1, j - 1)) && pv(1, j, j >= nb0);
          if (ok && j + 1 < nblk) ok = (DP == 64 || pv_over(1, j)) && qk(1, j + 1, j + 1 >= nb0);
        }
      } else {
        if (nblk > 0) ok = ok && qk(0, 0, true);
        for (int j = 0; ok && j < nblk; ++j) {
          if (j + 1 < nblk) ok = (j == 0 || pv_over(0, j - 1)) && qk(0, j + 1, true);
          if (ok) ok = pv(0, j, true);
        }
      }
      if (elect_one()) {
        tc_commit(drain);
        mbar_drain(drain, 0);
      }
      __syncwarp();
    } else {
      // ------------------------------------------------------------ V blocks at the end of what rows see
      const int tid = threadIdx.x - (kAux + 2) * 32;
      if (p.zero_unowned) attn_zero_unowned(p, false, blockIdx.x, gridDim.x, tid, 64);
      for (int e = 0; w.e0 + e < w.nblk; ++e) {
        const int j = w.e0 + e;
        if (!mbar_wait(&edge_full[e], 0, abort_flag, kDevErrWEmpty)) break;
        const int n = v_use<DP>(j, w.nblk), slot = n % Cfg::kSlots;
        uint4* blk = reinterpret_cast<uint4*>(ring + slot * U * kTileUnitBytes);
        bool odd = false;
        if (p.causal || j * kTileKeys + kTileKeys > s.nk) {
#pragma unroll 4
          for (int i = tid; i < U * 1024; i += 64) {
            const int key = j * kTileKeys + ((i & 1023) >> 3);   // the swizzle moves 16-byte chunks inside a row only
            if (key >= s.nk) {
              blk[i] = make_uint4(0, 0, 0, 0);
            } else if (p.causal) {
              uint4 x = blk[i];
              if (nonfinite2<BF16>(x.x) || nonfinite2<BF16>(x.y) || nonfinite2<BF16>(x.z) || nonfinite2<BF16>(x.w)) {
                x.x = finite2<BF16>(x.x); x.y = finite2<BF16>(x.y); x.z = finite2<BF16>(x.z); x.w = finite2<BF16>(x.w);
                blk[i] = x;
                odd = true;
              }
            }
          }
        }
        if (odd) *odd_values = 1;
        fence_proxy_async_shared();
        mbar_arrive(&edge_ready[e]);
      }
    }
  } else {
    // -------------------------------------------------------------- softmax: one thread per row
    if constexpr (kTwo) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(Cfg::kSoftmaxRegs));
    const int t = warp >> 2;
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const int row = (warp & 3) * 32 + lane;   // of the tile
    const int tok = w.t0 + t * tg.tokens + row / p.G, head = w.kvh * p.G + row % p.G;
    const bool real = row < tg.tokens * p.G && tok < s.nq;
    const int limit = !real ? -1 : p.causal ? min(s.nk - 1, tok + off) : s.nk - 1;   // last key this row sees
    // of the warp's first row, the least of its real rows
    const int limit0 = p.causal ? min(s.nk - 1, w.t0 + t * tg.tokens + (row - lane) / p.G + off) : s.nk - 1;
    const float sc = p.scale_log2;
    const float grow = 8.f / sc;
    float m = -INFINITY, l = 0.f;
    bool ok = t < w.ntile;
    const int nb = w.nb[t];
    for (int j = 0; ok && j < nb; ++j) {
      const int b = kTwo ? t : (j & 1);
      ok = __all_sync(0xffffffffu, mbar_wait(&s_full[b], kTwo ? (j & 1) : ((j >> 1) & 1), abort_flag, kDevErrAccFull));
      if (!ok) break;
      tc_fence_after();
      uint32_t v[4][32];
#pragma unroll
      for (int c = 0; c < 4; ++c) tmem_ld_32x32b_x32(tmem + lanes + Cfg::s_col(b) + c * 32, v[c]);
      tc_wait_ld();
      if (mode & kTileZeroScale) {
#pragma unroll
        for (int c = 0; c < 4; ++c)
#pragma unroll
          for (int i = 0; i < 32; ++i) v[c][i] = __float_as_uint(__uint_as_float(v[c][i]) * 0.f);
      }
      const bool edge = j * kTileKeys + kTileKeys - 1 > limit0;   // some row of the warp does not see all
      if (edge) {
        const int seen = limit - j * kTileKeys;
#pragma unroll
        for (int c = 0; c < 4; ++c)
#pragma unroll
          for (int i = 0; i < 32; ++i)
            if (c * 32 + i > seen) v[c][i] = 0xff800000u;
      }
      float mx[4];
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        mx[c] = m;
#pragma unroll
        for (int i = 0; i < 32; i += 2) mx[c] = max3(mx[c], __uint_as_float(v[c][i]), __uint_as_float(v[c][i + 1]));
      }
      const float top = max3(mx[0], mx[1], fmaxf(mx[2], mx[3]));
      if (j == 0) {
        m = top;
      } else {
        const bool need = top - m > grow;
        if (__any_sync(0xffffffffu, need)) {
          // scale what is accumulated; the product that adds to it is done first
          ok = __all_sync(0xffffffffu, mbar_wait(&pv_done[t], (j - 1) & 1, abort_flag, kDevErrAccEmpty));
          if (!ok) break;
          tc_fence_after();
          const float f = need ? ex2((m - top) * sc) : 1.f;
          if (need) m = top;
          l *= f;
#pragma unroll 1
          for (int c = 0; c < DP / 32; ++c) {
            uint32_t o[32];
            tmem_ld_32x32b_x32(tmem + lanes + Cfg::o_col(t) + c * 32, o);
            tc_wait_ld();
#pragma unroll
            for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
            tmem_st_32x32b_x32(tmem + lanes + Cfg::o_col(t) + c * 32, o);
          }
        }
      }
      const float bias = m == -INFINITY ? 0.f : -m * sc;
      const uint64_t sc2 = f2_pack(sc, sc), bias2 = f2_pack(bias, bias);
      // (a polynomial on the FMA pipe for 2 of every 16 pairs, to relieve the exponential unit, lengthened the
      // chain: 3.52 ms against 3.44 at 16384 tokens, 32 heads of 128)
      uint64_t sum = 0;   // (0.f, 0.f)
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        uint32_t pk[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const uint64_t x = f2_fma(f2_pack(__uint_as_float(v[c][2 * i]), __uint_as_float(v[c][2 * i + 1])), sc2, bias2);
          float p0, p1;
          f2_unpack(x, p0, p1);
          p0 = ex2(p0);
          p1 = ex2(p1);
          sum = f2_add(sum, f2_pack(p0, p1));
          pk[i] = pack2_rn<BF16>(p0, p1);
        }
        tmem_st_32x32b_x16(tmem + lanes + Cfg::p_col(b) + c * 16, pk);
        if (c >= 2) {   // 96 keys' weights: the product starts; then the rest
          tc_wait_st();
          tc_fence_before();
          // The last product starts with this arrival: the one before it is seen to be done first, or its phase
          // of pv_done could pass for the last one's below, or be over before it is looked at.
          if (c == 3 && j > 0 && j == nb - 1)
            ok = __all_sync(0xffffffffu, mbar_wait(&pv_done[t], (j - 1) & 1, abort_flag, kDevErrAccEmpty));
          mbar_arrive(c == 3 ? &p_full[b] : &p_part[b]);
        }
      }
      float s0, s1;
      f2_unpack(sum, s0, s1);
      l += s0 + s1;
    }
    // the row's output
    if (ok && nb > 0) ok = mbar_wait(&pv_done[t], (nb - 1) & 1, abort_flag, kDevErrAccEmpty);
    ok = __all_sync(0xffffffffu, ok);
    if (ok) {
      tc_fence_after();
      const bool odd = *odd_values != 0;
      const bool direct = tg.splits == 1;
      const float inv = direct ? attn_inverse(l, limit >= 0) : 1.f;
      uint16_t* dst = p.out + (long long)(s.q0 + tok) * p.o_st + head * p.o_sh;
      float* part = direct ? nullptr : tg.part + ((long long)blockIdx.x * Cfg::kTiles + t) * (128 * (DP + 2)) + row;
#pragma unroll 1
      for (int c = 0; c < DP / 32; ++c) {
        uint32_t o[32];
        if (nb > 0) {
          tmem_ld_32x32b_x32(tmem + lanes + Cfg::o_col(t) + c * 32, o);
          tc_wait_ld();
        } else {
#pragma unroll
          for (int i = 0; i < 32; ++i) o[i] = 0u;
        }
        if (real) {
          if (odd) {   // add the values that were taken out, where this row sees them
            for (int key = w.e0 * kTileKeys; key <= min(limit, w.nblk * kTileKeys - 1); ++key) {
              const uint16_t* vr = p.v + (long long)(s.k0 + key) * p.v_st + w.kvh * p.v_sh + c * 32;
#pragma unroll
              for (int i = 0; i < 32; ++i)
                if (c * 32 + i < p.D && nonfinite2<BF16>(vr[i]))
                  o[i] = __float_as_uint(__uint_as_float(o[i]) + bits_to_f32(vr[i], BF16 ? kBF16 : kF16));
            }
          }
          if (direct) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
              if (c * 32 + i * 8 < p.D) {
                uint4 x;
                x.x = pack2_rn<BF16>(__uint_as_float(o[8 * i]) * inv, __uint_as_float(o[8 * i + 1]) * inv);
                x.y = pack2_rn<BF16>(__uint_as_float(o[8 * i + 2]) * inv, __uint_as_float(o[8 * i + 3]) * inv);
                x.z = pack2_rn<BF16>(__uint_as_float(o[8 * i + 4]) * inv, __uint_as_float(o[8 * i + 5]) * inv);
                x.w = pack2_rn<BF16>(__uint_as_float(o[8 * i + 6]) * inv, __uint_as_float(o[8 * i + 7]) * inv);
                *reinterpret_cast<uint4*>(dst + c * 32 + i * 8) = x;
              }
          } else {
#pragma unroll
            for (int i = 0; i < 32; ++i) part[(c * 32 + i) * 128] = __uint_as_float(o[i]);
          }
        }
      }
      if (!direct && real) {
        part[DP * 128] = m * sc;
        part[(DP + 1) * 128] = l;
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == kAux + 1) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// Joins the parts of the keys, in order: a lane per row, a warp per 8 columns. Grid: units x tiles, 4 groups of 32
// rows, DP / 64 groups of columns.
template <bool BF16, int DP>
__global__ void __launch_bounds__(256) attn_tile_join_kernel(const AttnParams p, const TileGrid tg) {
  using Cfg = TileCfg<DP>;
  constexpr int kV = 8;   // columns of a thread
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int unit = blockIdx.x / Cfg::kTiles, t = blockIdx.x - unit * Cfg::kTiles;
  const int row = blockIdx.y * 32 + lane_id(), col = blockIdx.z * 64 + warp_id() * kV;
  const int kvh = unit / tg.slots;
  TileWork w;
  if (!tile_range<DP>(p, tg, tg.slots - 1 - (unit - kvh * tg.slots), w) || row >= tg.tokens * p.G) return;
  const int tok = w.t0 + t * tg.tokens + row / p.G;
  if (tok >= w.s.nq || col >= p.D) return;
  auto part = [&](int z) {
    return tg.part + (((long long)unit * tg.splits + z) * Cfg::kTiles + t) * (128 * (DP + 2)) + row;
  };
  if (part(0)[(DP + 1) * 128] < 0.f) return;   // nothing was run
  float mx = -INFINITY;
#pragma unroll 4
  for (int z = 0; z < tg.splits; ++z) mx = fmaxf(mx, part(z)[DP * 128]);
  const float ref = mx == -INFINITY ? 0.f : mx;
  float l = 0.f, acc[kV];
#pragma unroll
  for (int i = 0; i < kV; ++i) acc[i] = 0.f;
#pragma unroll 4
  for (int z = 0; z < tg.splits; ++z) {
    const float* x = part(z);
    const float f = ex2(x[DP * 128] - ref);
    l += f * x[(DP + 1) * 128];
#pragma unroll
    for (int i = 0; i < kV; ++i) acc[i] += f * x[(col + i) * 128];
  }
  const float inv = attn_inverse(l, tok >= attn_first_seeing(p, w.s));
  uint16_t* dst = p.out + (long long)(w.s.q0 + tok) * p.o_st + (kvh * p.G + row % p.G) * p.o_sh + col;
  *reinterpret_cast<uint4*>(dst) =
      make_uint4(pack2_rn<BF16>(acc[0] * inv, acc[1] * inv), pack2_rn<BF16>(acc[2] * inv, acc[3] * inv),
                 pack2_rn<BF16>(acc[4] * inv, acc[5] * inv), pack2_rn<BF16>(acc[6] * inv, acc[7] * inv));
}

}  // namespace oc
