// Attention for few query rows per sequence: single tokens, short runs of tokens, short prompts.
//
// Bound by HBM: one pass over the keys and values. The (token, head) rows of one key head are packed
// into tiles of 16 rows, so a group of query heads shares every key it reads. The work of a call is
// the list of 64-key blocks of all (sequence, key head, row tile) items in order; the CTAs of one
// full wave take equal runs of that list, found on the device from the length tables, so ragged
// lengths and long caches spread over every SM without the host knowing a length. Inside a run four
// or eight warps take 16-key slices in turn, each through a private cp.async ring of K and V units (no
// CTA barrier while streaming; TMA boxes of 16 keys, issued by the warps or by a warp of their own, took
// 146 and 176 us where these copies take 137: 48 tokens over caches up to 8192), with m16n8k16 tensor-core products, the running row maximum and sum in fp32 and base 2
// exponents. The warps are joined through shared memory; an item that spans CTAs leaves fp32
// partials (maximum, sum, unnormalized output) that attn_join_kernel adds in CTA order: no atomics,
// the same bits on every run.
#pragma once

#include "attn_common.cuh"

namespace oc {

constexpr int kSplitRows = 16;      // rows of a tile
constexpr int kSplitBlock = 64;     // keys of a work unit
constexpr int kSplitDescInts = 8;

template <int DP> struct SplitCfg {
  static constexpr int kWarps = DP == 256 ? 8 : 4;
  static constexpr int kThreads = kWarps * 32;
  static constexpr int kUnitBytes = 16 * DP * 2;               // 16 keys, or their values
  static constexpr int kUnits = DP == 256 ? 3 : DP == 128 ? 6 : 12;   // of a warp's ring: K, V, K, V, ...
  static constexpr int kCtasPerSm = DP == 256 ? 1 : 2;
  static constexpr int kRingBytes = kWarps * kUnits * kUnitBytes;   // 96 KB; 192 KB at DP = 256
  static constexpr int kPitch = DP + 8;                        // floats of a joined row
  static constexpr int kPartFloats = kSplitRows * (DP + 2);    // one partial: O [16][DP], m [16], l [16]
  static_assert(kWarps * kSplitRows * kPitch * 4 <= kRingBytes, "the warps' outputs fit the ring");
};

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool valid) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(valid ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void ldsm_x4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldsm_x4_trans(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
template <bool BF16>
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (BF16)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Work units of a sequence: key heads x row tiles x 64-key blocks (one block where no key is).
__device__ __forceinline__ int split_blocks(int nk) { return nk > 0 ? (nk + kSplitBlock - 1) / kSplitBlock : 1; }
__device__ __forceinline__ long long split_tiles(const AttnParams& p, int nq) {
  return ((long long)nq * p.G + kSplitRows - 1) / kSplitRows;
}
__device__ __forceinline__ long long split_units(const AttnParams& p, const Seq& s) {
  return (long long)p.Hkv * split_tiles(p, s.nq) * split_blocks(s.nk);
}

template <bool BF16, int DP>
__global__ void __launch_bounds__(SplitCfg<DP>::kThreads, SplitCfg<DP>::kCtasPerSm) attn_split_kernel(const AttnParams p) {
  using Cfg = SplitCfg<DP>;
  extern __shared__ __align__(128) uint8_t smem[];
  constexpr int kWarps = Cfg::kWarps;
  __shared__ float sm_m[kWarps][kSplitRows], sm_l[kWarps][kSplitRows];
  __shared__ int sm_odd;   // an infinity or NaN was taken out of the item's values
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int warp = warp_id(), lane = lane_id();
  const int g = lane >> 2, tq = lane & 3;
  int* desc = p.desc + blockIdx.x * kSplitDescInts;
  if (threadIdx.x == 0) {
    sm_odd = 0;
    desc[0] = 0;   // rows of the item this CTA begins and others finish
  }
  __syncthreads();

  // the call's units, then this CTA's run of them (every warp finds it for itself; with up to 32
  // sequences the tables are read once)
  long long total = 0, mine = 0;
  bool none = false;   // the table decreases: nothing is run
  for (int base = 0; base < p.B; base += 32) {
    Seq x{};
    if (base + lane < p.B) x = attn_seq(p, base + lane, blockIdx.x == 0 && warp == 0);
    mine = base + lane < p.B ? split_units(p, x) : 0;
    none |= __any_sync(0xffffffffu, x.down);
    long long sum = mine;
#pragma unroll
    for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    total += sum;
  }
  if (none) total = 0;
  if (p.zero_unowned) attn_zero_unowned(p, none, blockIdx.x, gridDim.x, threadIdx.x, Cfg::kThreads);
  const int busy = (int)min(total, (long long)gridDim.x);   // CTAs with work
  if ((int)blockIdx.x >= busy) return;
  long long u, u_end;
  if (total < (1ll << 22)) {   // the grid is below 2^10: 32-bit divisions
    u = (unsigned)total * blockIdx.x / (unsigned)busy;
    u_end = (unsigned)total * (blockIdx.x + 1) / (unsigned)busy;
  } else {
    u = total * blockIdx.x / busy;
    u_end = total * (blockIdx.x + 1) / busy;
  }
  int b = 0;
  long long seq_begin = 0;   // first unit of sequence b
  for (int base = 0; base < p.B; base += 32) {
    if (p.B > 32) mine = base + lane < p.B ? split_units(p, attn_seq(p, base + lane)) : 0;
    long long incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long y = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += y;
    }
    const unsigned past = __ballot_sync(0xffffffffu, base + lane < p.B && seq_begin + incl > u);
    if (past) {
      const int f = __ffs(past) - 1;
      b = base + f;
      seq_begin += __shfl_sync(0xffffffffu, incl - mine, f);
      break;
    }
    seq_begin += __shfl_sync(0xffffffffu, incl, 31);
  }
  Seq s = attn_seq(p, b);

  uint8_t* ring = smem + warp * (Cfg::kUnits * Cfg::kUnitBytes);
  const uint32_t ring_addr = smem_u32(ring);
  constexpr int kCh = DP / 8;                      // 16-byte chunks of a row
  constexpr int kIter = 16 * kCh / 32;             // chunks per lane of one 16-row matrix
  constexpr int kStep = 32 / kCh;                  // rows from one of a lane's chunks to its next

  while (u < u_end) {
    while (u >= seq_begin + split_units(p, s)) {
      seq_begin += split_units(p, s);
      s = attn_seq(p, ++b);
    }
    const int nblk = split_blocks(s.nk);
    const long long rel = u - seq_begin;
    const long long item = rel < (1ll << 31) ? (long long)((unsigned)rel / (unsigned)nblk) : rel / nblk;
    const int blk0 = (int)(rel - item * nblk);
    const int blk1 = (int)min((long long)nblk, blk0 + (u_end - u));
    const long long tiles = split_tiles(p, s.nq);
    const int kvh = (item | tiles) < (1ll << 31) ? (int)((unsigned)item / (unsigned)tiles) : (int)(item / tiles);
    const long long row0 = (item - kvh * tiles) * kSplitRows;
    const int rows = (int)min((long long)kSplitRows, (long long)s.nq * p.G - row0);
    const int kbeg = blk0 * kSplitBlock, kend = min(s.nk, blk1 * kSplitBlock);

    float o[DP / 8][4];
#pragma unroll
    for (int i = 0; i < DP / 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};

    const uint16_t* kb = p.k + s.k0 * p.k_st + kvh * p.k_sh;
    const uint16_t* vb = p.v + s.k0 * p.v_st + kvh * p.v_sh;
    const int slices = kend > kbeg ? (kend - kbeg + 15) / 16 : 0;
    // rows behind the last key and columns behind D are filled with zeros: a weight of zero times
    // whatever lies there must not reach the output
    const int c_row = lane / kCh, c_ch = lane % kCh;
    const bool c_in = c_ch * 8 < p.D;
    const uint16_t* k_src = kb + (long long)(kbeg + c_row) * p.k_st + c_ch * 8;
    const uint16_t* v_src = vb + (long long)(kbeg + c_row) * p.v_st + c_ch * 8;
    // the warp's unit n of this item: K (even) or V (odd) of its slice n / 2, into ring place `at`
    const int units = (slices > warp ? (slices - warp + kWarps - 1) / kWarps : 0) * 2;
    auto issue = [&](int n, int at) {
      if (n < units) {
        const int sl = warp + (n >> 1) * kWarps;
        const long long st = n & 1 ? p.v_st : p.k_st;
        const uint16_t* src = (n & 1 ? v_src : k_src) + (long long)sl * 16 * st;
        const uint32_t dst = ring_addr + at * Cfg::kUnitBytes + c_row * (DP * 2);
        const int left = kend - kbeg - sl * 16 - c_row;   // rows this lane may still copy
        if (sl * 16 + 16 <= kend - kbeg && p.D == DP) {
#pragma unroll
          for (int i = 0; i < kIter; ++i) {
            cp_async16(dst + i * kStep * (DP * 2) + ((c_ch ^ ((i * kStep + c_row) & 7)) * 16), src);
            src += kStep * st;
          }
        } else {
#pragma unroll
          for (int i = 0; i < kIter; ++i) {
            const bool ok = c_in && i * kStep < left;
            cp_async16(dst + i * kStep * (DP * 2) + ((c_ch ^ ((i * kStep + c_row) & 7)) * 16), ok ? src : p.k, ok);
            src += kStep * st;
          }
        }
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
    };
    constexpr int NU = Cfg::kUnits;
#pragma unroll 1
    for (int i = 0; i < NU - 1; ++i) issue(i, i);

    // this lane's two rows: last visible key, and the queries as A fragments
    int limit[2];
    uint32_t qa[DP / 16][4];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int r = g + 8 * i;
      const long long row = row0 + r;
      const int tok = (int)(row / p.G);
      const uint16_t* qr = p.q + (s.q0 + tok) * p.q_st + (kvh * p.G + row % p.G) * p.q_sh + 2 * tq;
      limit[i] = r < rows ? (p.causal ? min(kend - 1, tok + s.nk - s.nq) : kend - 1) : -1;
#pragma unroll
      for (int ks = 0; ks < DP / 16; ++ks)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int col = ks * 16 + h * 8;
          qa[ks][2 * h + i] = (r < rows && col < p.D) ? *reinterpret_cast<const uint32_t*>(qr + col) : 0u;
        }
    }
    // slices from edge_begin on hold keys that some row of the tile does not see
    const int first_limit = p.causal ? (int)(row0 / p.G) + s.nk - s.nq : kend - 1;   // of the tile's first token
    const int edge_begin = kbeg + max(0, min(first_limit + 1, kend) - kbeg) / 16 * 16;
    const bool has_edge = first_limit < kend - 1;
    // ldmatrix addresses: 16-byte chunk c of a row lies at ((c ^ (row & 7)) * 16) of its 128-byte part, so step k of
    // a part's four flips bits of the lane's first address
    const int k_row = (lane & 7) + ((lane >> 4) << 3), v_row = lane & 15;
    const uint32_t k_at = ring_addr + k_row * (DP * 2) + ((((lane >> 3) & 1) ^ (k_row & 7)) << 4);
    const uint32_t v_at = ring_addr + v_row * (DP * 2) + (((lane >> 4) ^ (v_row & 7)) << 4);
    int place = 0;   // of the next unit to read; the one before it is refilled
    auto step = [&](int n) {   // unit n has landed, and the unit that was read last makes room
      asm volatile("cp.async.wait_group %0;" ::"n"(NU - 2) : "memory");
      __syncwarp();
      issue(n + NU - 1, place == 0 ? NU - 1 : place - 1);
      const int at = place;
      place = place + 1 == NU ? 0 : place + 1;
      return at;
    };
    for (int n = 0; n < units; n += 2) {
      const int sl = warp + (n >> 1) * kWarps;
      const uint32_t ks_addr = k_at + step(n) * Cfg::kUnitBytes;
      const int key0 = kbeg + sl * 16;
      float c[2][4] = {}, c2[2][4] = {};   // two chains each: the products of one sum wait for one another
#pragma unroll
      for (int ks = 0; ks < DP / 16; ++ks) {
        uint32_t r[4];
        ldsm_x4((ks_addr ^ ((ks & 3) << 5)) + (ks >> 2) * 128, r);
        mma16816<BF16>(ks & 1 ? c2[0] : c[0], qa[ks], r[0], r[1]);
        mma16816<BF16>(ks & 1 ? c2[1] : c[1], qa[ks], r[2], r[3]);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) { c[0][i] += c2[0][i]; c[1][i] += c2[1][i]; }
      // The exponents' reference follows the running maximum only when it grew by more than 2^8 (weights
      // up to 256 are as exact in 16 bits as weights up to 1): the output is rarely scaled.
      float top[2];
      bool grew = false;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        top[i] = m[i];
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float& x = c[t][2 * i + e];
            x = key0 + t * 8 + 2 * tq + e <= limit[i] ? x * p.scale_log2 : -INFINITY;
            top[i] = fmaxf(top[i], x);
          }
        top[i] = fmaxf(top[i], __shfl_xor_sync(0xffffffffu, top[i], 1));
        top[i] = fmaxf(top[i], __shfl_xor_sync(0xffffffffu, top[i], 2));
        grew |= top[i] - m[i] > 8.f;
      }
      if (__any_sync(0xffffffffu, grew)) {
        float corr[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          corr[i] = top[i] > m[i] ? ex2(m[i] - top[i]) : 1.f;
          m[i] = fmaxf(m[i], top[i]);
          l[i] *= corr[i];
        }
#pragma unroll
        for (int i = 0; i < DP / 8; ++i) {
          o[i][0] *= corr[0]; o[i][1] *= corr[0];
          o[i][2] *= corr[1]; o[i][3] *= corr[1];
        }
      }
      uint32_t pa[4];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float ref = m[i] == -INFINITY ? 0.f : m[i];
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          const float p0 = ex2(c[t][2 * i] - ref), p1 = ex2(c[t][2 * i + 1] - ref);
          l[i] += p0 + p1;
          pa[2 * t + i] = pack2_rn<BF16>(p0, p1);   // rounded once, as the product takes them; l adds them unrounded
        }
      }
      // A value that a row does not see may be infinite or NaN, and its weight of zero must not turn that
      // into NaN: such values leave the slice, and the rows that see them add them at the end.
      const int v_place = step(n + 1);
      const uint32_t vs_addr = v_at + v_place * Cfg::kUnitBytes;
      if (has_edge && key0 >= edge_begin) {
        uint4* vsl = reinterpret_cast<uint4*>(ring + v_place * Cfg::kUnitBytes);
#pragma unroll 1
        for (int i = lane; i < 16 * kCh; i += 32) {
          uint4 x = vsl[i];
          if (nonfinite2<BF16>(x.x) || nonfinite2<BF16>(x.y) || nonfinite2<BF16>(x.z) || nonfinite2<BF16>(x.w)) {
            vsl[i] = make_uint4(finite2<BF16>(x.x), finite2<BF16>(x.y), finite2<BF16>(x.z), finite2<BF16>(x.w));
            sm_odd = 1;
          }
        }
        __syncwarp();
      }
#pragma unroll
      for (int d2 = 0; d2 < DP / 16; ++d2) {
        uint32_t r[4];
        ldsm_x4_trans((vs_addr ^ ((d2 & 3) << 5)) + (d2 >> 2) * 128, r);
        mma16816<BF16>(o[2 * d2], pa, r[0], r[1]);
        mma16816<BF16>(o[2 * d2 + 1], pa, r[2], r[3]);
      }
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    __syncthreads();   // the rings are read; they now hold the warps' outputs

    float* osm = reinterpret_cast<float*>(smem);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      l[i] += __shfl_xor_sync(0xffffffffu, l[i], 1);
      l[i] += __shfl_xor_sync(0xffffffffu, l[i], 2);
      float* orow = osm + (warp * kSplitRows + g + 8 * i) * Cfg::kPitch;
#pragma unroll
      for (int d = 0; d < DP / 8; ++d)
        *reinterpret_cast<float2*>(orow + d * 8 + 2 * tq) = make_float2(o[d][2 * i], o[d][2 * i + 1]);
      if (tq == 0) {
        sm_m[warp][g + 8 * i] = m[i];
        sm_l[warp][g + 8 * i] = l[i];
      }
    }
    __syncthreads();
    const bool whole = blk0 == 0 && blk1 == nblk;
    float* part = p.part + ((long long)blockIdx.x * 2 + (blk0 == 0 ? 1 : 0)) * Cfg::kPartFloats;
    for (int i = threadIdx.x; i < rows * (DP / 4); i += Cfg::kThreads) {
      const int r = i / (DP / 4), c4 = (i % (DP / 4)) * 4;
      float mx = -INFINITY;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) mx = fmaxf(mx, sm_m[w][r]);
      const float ref = mx == -INFINITY ? 0.f : mx;
      float lsum = 0.f;
      float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float a = ex2(sm_m[w][r] - ref);
        const float4 x = *reinterpret_cast<const float4*>(osm + (w * kSplitRows + r) * Cfg::kPitch + c4);
        lsum += a * sm_l[w][r];
        acc.x += a * x.x; acc.y += a * x.y; acc.z += a * x.z; acc.w += a * x.w;
      }
      if (has_edge && sm_odd) {
        const int last = min(kend - 1, (int)((row0 + r) / p.G) + s.nk - s.nq);
        for (int key = edge_begin; key <= last; ++key) {
          const uint16_t* vr = vb + (long long)key * p.v_st + c4;
          float* y = &acc.x;
          for (int e = 0; e < 4; ++e)
            if (c4 < p.D && nonfinite2<BF16>(vr[e])) y[e] += bits_to_f32(vr[e], BF16 ? kBF16 : kF16);
        }
      }
      if (whole) {
        if (c4 < p.D) {
          const long long row = row0 + r;
          const float inv = attn_inverse(lsum, row / p.G >= attn_first_seeing(p, s));
          uint16_t* dst = p.out + (s.q0 + row / p.G) * p.o_st + (kvh * p.G + row % p.G) * p.o_sh + c4;
          *reinterpret_cast<uint2*>(dst) = make_uint2(pack2_rn<BF16>(acc.x * inv, acc.y * inv),
                                                      pack2_rn<BF16>(acc.z * inv, acc.w * inv));
        }
      } else {
        *reinterpret_cast<float4*>(part + r * DP + c4) = acc;
        if (c4 == 0) {
          part[kSplitRows * DP + r] = mx;
          part[kSplitRows * DP + kSplitRows + r] = lsum;
        }
      }
    }
    if (!whole && blk0 == 0 && threadIdx.x == 0) {
      const long long last = seq_begin + (item + 1) * nblk - 1;   // the item's last unit
      desc[1] = (int)(((last + 1) * busy - 1) / total);           // the CTA that holds it
      desc[2] = s.q0;
      desc[3] = kvh;
      *reinterpret_cast<long long*>(desc + 4) = row0;
      desc[6] = attn_first_seeing(p, s);
      desc[0] = rows;
    }
    __syncthreads();
    if (has_edge && threadIdx.x == 0) sm_odd = 0;   // read above, written again by the next item's slices
    if (has_edge) __syncthreads();
    u += blk1 - blk0;
  }
}

// Joins the partials of the item that CTA blockIdx.x began: slot 1 of that CTA, slot 0 of the CTAs
// after it up to the item's last one. Four rows to a block, four warps to a row, each of which takes
// every fourth partial in order: eight independent loads are in flight, and the sums' order is fixed.
constexpr int kJoinThreads = 512;
template <bool BF16, int DP>
__global__ void __launch_bounds__(kJoinThreads) attn_join_kernel(const AttnParams p) {
  using Cfg = SplitCfg<DP>;
  constexpr int kV = DP / 32;   // columns of a lane
  __shared__ float sm_acc[4][4][DP], sm_m[4][4], sm_l[4][4];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int* desc = p.desc + blockIdx.x * kSplitDescInts;
  if ((int)blockIdx.y * 4 >= desc[0]) return;
  const int row_in = warp_id() >> 2, part = warp_id() & 3, lane = lane_id();
  const int r = blockIdx.y * 4 + row_in;
  const int c0 = blockIdx.x, count = desc[1] - c0 + 1;
  auto slot = [&](int i) { return p.part + ((long long)(c0 + i) * 2 + (i == 0 ? 1 : 0)) * Cfg::kPartFloats; };
  float mx = -INFINITY, lsum = 0.f, acc[kV];
#pragma unroll
  for (int i = 0; i < kV; ++i) acc[i] = 0.f;
  // this warp's partials: part, part + 4, ...; a lane looks at one of up to 32 of them at a time
  const int mine = count > part ? (count - part + 3) / 4 : 0;
  for (int base = 0; base < mine; base += 32) {
    float m = -INFINITY, l = 0.f;
    if (base + lane < mine) {
      const float* ml = slot(part + 4 * (base + lane)) + kSplitRows * DP + r;
      m = ml[0];
      l = ml[kSplitRows];
    }
    float top = fmaxf(mx, m);
#pragma unroll
    for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    const float ref = top == -INFINITY ? 0.f : top;
    const float old = ex2(mx - ref), w = ex2(m - ref);
    mx = top;
    float sum = w * l;
#pragma unroll
    for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    lsum = lsum * old + sum;
#pragma unroll
    for (int i = 0; i < kV; ++i) acc[i] *= old;
    const int here = min(32, mine - base);
#pragma unroll 8
    for (int i = 0; i < here; ++i) {
      const float a = __shfl_sync(0xffffffffu, w, i);
      const float* src = slot(part + 4 * (base + i)) + r * DP + lane * kV;
#pragma unroll
      for (int e = 0; e < kV; ++e) acc[e] += a * src[e];
    }
  }
#pragma unroll
  for (int e = 0; e < kV; ++e) sm_acc[row_in][part][lane * kV + e] = acc[e];
  if (lane == 0) {
    sm_m[row_in][part] = mx;
    sm_l[row_in][part] = lsum;
  }
  __syncthreads();
  if (part != 0 || r >= desc[0]) return;
  float top = -INFINITY, total = 0.f, f[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) top = fmaxf(top, sm_m[row_in][i]);
  const float ref = top == -INFINITY ? 0.f : top;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f[i] = ex2(sm_m[row_in][i] - ref);
    total += f[i] * sm_l[row_in][i];
  }
  const long long row = *reinterpret_cast<const long long*>(desc + 4) + r;
  const float inv = attn_inverse(total, row / p.G >= desc[6]);
  uint16_t* dst = p.out + (desc[2] + row / p.G) * p.o_st + (desc[3] * p.G + row % p.G) * p.o_sh + lane * kV;
  if (lane * kV < p.D) {
#pragma unroll
    for (int e = 0; e < kV; e += 2) {
      float x[2] = {0.f, 0.f};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        x[0] += f[i] * sm_acc[row_in][i][lane * kV + e];
        x[1] += f[i] * sm_acc[row_in][i][lane * kV + e + 1];
      }
      *reinterpret_cast<uint32_t*>(dst + e) = pack2_rn<BF16>(x[0] * inv, x[1] * inv);
    }
  }
}

}  // namespace oc
