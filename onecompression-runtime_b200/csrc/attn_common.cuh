// Attention over packed sequences: what the kernels share.
//
// Sequence b owns the query rows [cu_q[b], cu_q[b+1]) and the key rows that start at cu_k[b]; it
// sees kv_lens[b] of them, or all up to cu_k[b+1]. With causal masking the last query sees the last
// key: query i of nq sees the keys j <= i + nk - nq. A row that sees no key gives zeros; a row whose
// visible scores are all minus infinity gives NaN, as its softmax does.
// The tables live on the device and are clamped to the tensors here, so no table value can send an
// access out of range; a clamped value sets the device error word. A query table that decreases sets it
// too, and no sequence of it is run: rows would have several owners, or none.
#pragma once

#include "common.cuh"

namespace oc {

struct AttnParams {
  const uint16_t* q;
  const uint16_t* k;
  const uint16_t* v;
  uint16_t* out;
  long long q_st, q_sh, k_st, k_sh, v_st, v_sh, o_st, o_sh;  // token and head strides (elements)
  int Tq, Tk, Hq, Hkv, G, D;                                 // G = Hq / Hkv
  const int* cu_q;      // [B + 1] or null: one sequence over all rows
  const int* cu_k;
  const int* kv_lens;   // [B] or null
  int B;
  int causal;
  int zero_unowned;     // also write zeros to the query rows that no sequence owns
  float scale_log2;     // softmax scale * log2(e)
  float* part;          // split kernel: partial results
  int* desc;            // split kernel: one descriptor per CTA
};

struct Seq {
  int q0, nq, k0, nk;
  bool down;   // the query table decreases here
};

// The first token of a sequence that sees a key (nq where none does).
__device__ __forceinline__ int attn_first_seeing(const AttnParams& p, const Seq& s) {
  return p.causal ? max(0, s.nq - s.nk) : s.nk > 0 ? 0 : s.nq;
}
// What the sum of weighted values is multiplied with, from the sum of weights. The key with the largest score
// weighs at least 1, so a sum of zero means no key, or no score above minus infinity.
__device__ __forceinline__ float attn_inverse(float l, bool sees_keys) {
  return l > 0.f ? 1.f / l : l == 0.f ? (sees_keys ? __int_as_float(0x7fffffff) : 0.f) : l;
}

__device__ __forceinline__ Seq attn_seq(const AttnParams& p, int b, bool report = false) {
  int q0 = 0, q1 = p.Tq, k0 = 0, k1 = p.Tk;
  if (p.cu_q) { q0 = p.cu_q[b]; q1 = p.cu_q[b + 1]; }
  if (p.cu_k) { k0 = p.cu_k[b]; k1 = p.cu_k[b + 1]; }
  Seq s;
  s.q0 = min(max(q0, 0), p.Tq);
  const int qe = min(max(q1, s.q0), p.Tq);
  s.k0 = min(max(k0, 0), p.Tk);
  const int ke = min(max(k1, s.k0), p.Tk);
  s.nq = qe - s.q0;
  s.down = q1 < q0;
  s.nk = ke - s.k0;
  bool bad = s.q0 != q0 || qe != q1 || s.k0 != k0 || ke != k1;
  if (p.kv_lens) {
    const int n = p.kv_lens[b];
    bad |= n < 0 || n > s.nk;
    s.nk = min(max(n, 0), s.nk);
  }
  if (report && bad) record_error(kDevErrSeq);
  return s;
}

// Does the query table decrease at one of the places that this thread of `threads` looks at?
__device__ __forceinline__ bool attn_disorder(const AttnParams& p, int tid, int threads) {
  bool down = false;
  if (p.cu_q)
#pragma unroll 4
    for (int b = tid; b < p.B; b += threads) down |= p.cu_q[b + 1] < p.cu_q[b];
  return down;
}

// One CTA's share of the rows that no sequence owns, in front of the first one and behind the last (all of
// them without sequences, or where `none` is run): zeros (D is a multiple of 8, rows 16-byte aligned). By
// `threads` threads of the CTA, of which this is `tid`.
__device__ __forceinline__ void attn_zero_unowned(const AttnParams& p, bool none, int cta, int n_ctas, int tid,
                                                  int threads) {
  if (!p.cu_q) return;
  const int vecs = p.D / 8;
  const int head = p.B > 0 ? min(max(p.cu_q[0], 0), p.Tq) : 0;
  const int tail = p.B > 0 && !none ? min(max(p.cu_q[p.B], head), p.Tq) : head;
  const long long rows = (long long)head + (p.Tq - tail);
  for (long long r = cta; r < rows; r += n_ctas) {
    const long long t = r < head ? r : tail + (r - head);
    for (long long i = tid; i < (long long)p.Hq * vecs; i += threads)   // up to 2^35
      *reinterpret_cast<uint4*>(p.out + t * p.o_st + (i / vecs) * p.o_sh + (i % vecs) * 8) = make_uint4(0, 0, 0, 0);
  }
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Pairs of fp32 values in one 64-bit register (the FMA pipe takes both halves in one issue slot).
__device__ __forceinline__ uint64_t f2_pack(float lo, float hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ void f2_unpack(uint64_t v, float& lo, float& hi) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v));
}
__device__ __forceinline__ uint64_t f2_fma(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ uint64_t f2_add(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// Is one of the two 16-bit values of a register infinite or NaN?
template <bool BF16> __device__ __forceinline__ bool nonfinite2(uint32_t v) {
  constexpr uint32_t m = BF16 ? 0x7F80u : 0x7C00u;
  return (v & m) == m || ((v >> 16) & m) == m;
}
// The register with infinite and NaN halves set to zero.
template <bool BF16> __device__ __forceinline__ uint32_t finite2(uint32_t v) {
  constexpr uint32_t m = BF16 ? 0x7F80u : 0x7C00u;
  if ((v & m) == m) v &= 0xFFFF0000u;
  if (((v >> 16) & m) == m) v &= 0x0000FFFFu;
  return v;
}

}  // namespace oc
