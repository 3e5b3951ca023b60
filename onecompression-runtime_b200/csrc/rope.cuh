// Rotary positions: every rotated pair (x1, x2) of a head becomes
//   y1 = g (x1 cos a - x2 sin a),  y2 = g (x2 cos a + x1 sin a),  a = position * f_pair.
//
// Angles: f_pair is kept as the fraction of a turn per position, a 0.64 fixed-point number, so
// position * fraction modulo 2^64 (one integer product, wrapping) is the angle modulo one turn, for
// every 64-bit position, negative ones included. Its upper 32 bits as a signed number are the angle in
// half turns x 2^31, which sincospif takes without a range reduction. The error is 2^-25 of a half turn
// (the conversion to fp32) plus the position times what the table is off (2^-64 of a half turn at least);
// an fp32 product would lose the angle of far positions.
//
// Bound by HBM: each value is read and written once. A block takes TB tokens, computes their
// TB * R/2 sines and cosines once into shared memory (all heads of a token share them) and then
// walks the heads, one unit of two 16-byte vectors (V pairs) per thread and two units in flight.
#pragma once

#include "common.cuh"

namespace oc {

struct RopeTensor {
  const void* x;
  void* y;
  long long xst, xsh, yst, ysh;  // token and head strides (elements)
  int H;
};

struct RopeParams {
  RopeTensor t[2];
  int T, D, R;
  const void* pos;       // [T, A] int32 or int64, rows pos_st apart
  int pos64;
  long long pos_st;
  const unsigned long long* turns;  // [R/2]
  const uint8_t* axis;              // [R/2] or null (one axis)
  float gain;
  int heads_per_block;   // of the Hq + Hk heads
  int copy_rest;         // out of place: the D - R values behind the rotated part are copied
};

constexpr int kRopeThreads = 256;

template <int DT> struct RopeElem;
template <> struct RopeElem<kF16> {
  using T = uint16_t;
  __device__ static float get(T b) { return __half2float(__ushort_as_half(b)); }
  __device__ static T put(float v) { return __half_as_ushort(__float2half_rn(v)); }
};
template <> struct RopeElem<kBF16> {
  using T = uint16_t;
  __device__ static float get(T b) { return __bfloat162float(__ushort_as_bfloat16(b)); }
  __device__ static T put(float v) { return __bfloat16_as_ushort(__float2bfloat16_rn(v)); }
};
template <> struct RopeElem<kF32> {
  using T = float;
  __device__ static float get(T b) { return b; }
  __device__ static T put(float v) { return v; }
};

// V values per vector: 16 bytes, or 1 where sizes, strides or pointers do not allow vectors.
template <int DT, int V, bool INTER, int TB>
__global__ void __launch_bounds__(kRopeThreads, 4) rope_kernel(const RopeParams p) {
  using El = RopeElem<DT>;
  using E = typename El::T;
  struct alignas(sizeof(E) * V) Vec { E e[V]; };
  extern __shared__ float rope_smem[];
  const int P = p.R / 2;
  float* cs = rope_smem;            // [TB][P]
  float* sn = rope_smem + TB * P;
  const int t0 = blockIdx.x * TB;
  const int nt = min(TB, p.T - t0);
  for (int i = threadIdx.x; i < nt * P; i += kRopeThreads) {
    const int t = i / P, pr = i - t * P;
    const long long at = (long long)(t0 + t) * p.pos_st + (p.axis ? p.axis[pr] : 0);
    const long long pos = p.pos64 ? reinterpret_cast<const long long*>(p.pos)[at]
                                  : (long long)reinterpret_cast<const int*>(p.pos)[at];
    const unsigned long long a = (unsigned long long)pos * p.turns[pr];
    float s, c;
    sincospif((float)(int)(unsigned)(a >> 32) * 0x1p-31f, &s, &c);
    cs[i] = c * p.gain;
    sn[i] = s * p.gain;
  }
  __syncthreads();

  const int UR = P / V;                                         // rotated units of a head
  const int U = UR + (p.copy_rest ? (p.D - p.R) / (2 * V) : 0);
  const int h_begin = blockIdx.y * p.heads_per_block;
  const int nh = min(p.heads_per_block, p.t[0].H + p.t[1].H - h_begin);
  // a thread keeps its unit and walks (token, head) in steps of the heads that the block covers at once
  const int width = min(U, kRopeThreads), rows = kRopeThreads / width;
  const int hr = threadIdx.x / width;
  if (hr >= min(rows, nh)) return;
  constexpr int kBatch = 2;
  for (int u = threadIdx.x - hr * width; u < U; u += width) {
    const bool rot = u < UR;
    const int col = rot ? (INTER ? 2 * u * V : u * V) : p.R + (u - UR) * 2 * V;
    const int second = rot && !INTER ? P : V;   // distance of the pair's second vector
    int t = 0, h = hr;
    while (t < nt) {
      Vec a[kBatch], b[kBatch];
      E* dst[kBatch];
      int trig[kBatch];
#pragma unroll
      for (int j = 0; j < kBatch; ++j) {
        dst[j] = nullptr;
        if (t < nt) {
          const int hh = h_begin + h;
          const bool is_k = hh >= p.t[0].H;
          const RopeTensor& x = p.t[is_k ? 1 : 0];
          const long long hx = is_k ? hh - p.t[0].H : hh;
          const E* src = reinterpret_cast<const E*>(x.x) + (t0 + t) * x.xst + hx * x.xsh + col;
          dst[j] = reinterpret_cast<E*>(x.y) + (t0 + t) * x.yst + hx * x.ysh + col;
          trig[j] = t * P + u * V;
          a[j] = *reinterpret_cast<const Vec*>(src);
          b[j] = *reinterpret_cast<const Vec*>(src + second);
          h += rows;
          if (h >= nh) { h = hr; ++t; }
        }
      }
#pragma unroll
      for (int j = 0; j < kBatch; ++j) {
        if (!dst[j]) continue;
        if (rot) {
          const float* c = cs + trig[j];
          const float* s = sn + trig[j];
#pragma unroll
          for (int e = 0; e < V; ++e) {
            // half layout: pair e is (a[e], b[e]); interleaved: neighbours of the 2V values a, b
            E& e1 = INTER ? (2 * e < V ? a[j].e[(2 * e) % V] : b[j].e[(2 * e) % V]) : a[j].e[e];
            E& e2 = INTER ? (2 * e + 1 < V ? a[j].e[(2 * e + 1) % V] : b[j].e[(2 * e + 1) % V]) : b[j].e[e];
            const float x1 = El::get(e1), x2 = El::get(e2);
            e1 = El::put(x1 * c[e] - x2 * s[e]);
            e2 = El::put(x2 * c[e] + x1 * s[e]);
          }
        }
        *reinterpret_cast<Vec*>(dst[j]) = a[j];
        *reinterpret_cast<Vec*>(dst[j] + second) = b[j];
      }
    }
  }
}

}  // namespace oc
