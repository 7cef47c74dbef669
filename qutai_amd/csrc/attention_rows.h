// One wave per row: attention for any head dimension up to 256, fp32 or bf16
// storage of any alignment, fp32 math (the reference's warp kernels
// lm_attention / lm_attention_delta / lm_attention_backward_q / _kv,
// src/qutai/backends/cuda/lm.cu:65-87 and :289-343).  One wave computes a
// query row (forward, dq) or key row (dk, dv); lane l owns dimensions l,
// l + 64, l + 128, l + 192; dot products are wave-wide sums.  Bound by the
// cross-lane sums of every score, so it serves the rows that the matrix
// kernels (attention_mma.h) leave: rows that are not 16-byte aligned,
// sequences of a few positions, and waves whose operands hold an infinity or
// a NaN.
#pragma once
#include "attention_common.h"

namespace {

struct AttnGenArgs {
  const void* g;
  const void* q;
  const void* k;
  const void* v;
  const void* o;
  float* lse;
  float* delta;
  void* dq;  // forward: the output
  void* dk;
  void* dv;
  int64_t batch, heads, kv_heads, time, dim;
  int64_t qb, qh, qt, kb, kh, kt, lb, lh, lt;
  float scale;
  float scale_log2, scale_log2_lo;  // scale * log2(e) and its rounding error
  int causal;
  // split: each dK/dV workgroup takes one query head of its kv head's group
  // and writes unscaled fp32 partials to part_k / part_v + head * part_stride
  // (dk's element offsets); dkv_sum adds them up
  int split;
  float* part_k;
  float* part_v;
  int64_t part_stride;
};

// Sequences of different lengths, one behind the other in rows of tokens (b = 0):
// of a workgroup's tile the tables hold its sequence's start with the tile's first
// row in it (32 bits up) and the sequence's length, and q, k, v and their gradients may
// be columns of wider matrices.
struct AttnPackedArgs : AttnGenArgs {
  const int64_t* tiles;
  const int64_t* lengths;
  int64_t vt, ot, dqt, dkt, dvt;  // elements from row to row of v, of out and its gradient, and of dq, dk, dv
  void* rest;                     // what out's rounding left, or null
  int pack;                       // query heads of a kv head that share a workgroup
};

// Elements from row to row, where a packed call's differ from the others'.
__device__ __forceinline__ int64_t value_pitch(const AttnGenArgs& p) { return p.kt; }
__device__ __forceinline__ int64_t out_pitch(const AttnGenArgs& p) { return p.qt; }
__device__ __forceinline__ int64_t dq_pitch(const AttnGenArgs& p) { return p.qt; }
__device__ __forceinline__ int64_t dk_pitch(const AttnGenArgs& p) { return p.kt; }
__device__ __forceinline__ int64_t dv_pitch(const AttnGenArgs& p) { return p.kt; }
__device__ __forceinline__ int64_t part_pitch(const AttnGenArgs& p) { return p.kt; }
__device__ __forceinline__ int64_t value_pitch(const AttnPackedArgs& p) { return p.vt; }
__device__ __forceinline__ int64_t out_pitch(const AttnPackedArgs& p) { return p.ot; }
__device__ __forceinline__ int64_t dq_pitch(const AttnPackedArgs& p) { return p.dqt; }
__device__ __forceinline__ int64_t dk_pitch(const AttnPackedArgs& p) { return p.dkt; }
__device__ __forceinline__ int64_t dv_pitch(const AttnPackedArgs& p) { return p.dvt; }
__device__ __forceinline__ int64_t part_pitch(const AttnPackedArgs& p) { return p.kv_heads * p.dim; }

// The arguments of tile `tile`'s sequence alone; returns the tile's first row in it.
template <class T>
__device__ __forceinline__ int enter_sequence(AttnPackedArgs& p, int64_t tile) {
  const int64_t word = uniform64(p.tiles[tile]), start = word & 0xffffffff;
  p.time = uniform64(p.lengths[tile]);
  const auto at = [&](const void* x, int64_t pitch) { return (const void*)((const T*)x + start * pitch); };
  p.q = at(p.q, p.qt);
  p.k = at(p.k, p.kt);
  p.v = at(p.v, p.vt);
  p.g = at(p.g, p.ot);
  p.o = at(p.o, p.ot);
  p.dq = const_cast<void*>(at(p.dq, p.dqt));
  p.dk = const_cast<void*>(at(p.dk, p.dkt));
  p.dv = const_cast<void*>(at(p.dv, p.dvt));
  if (p.rest) p.rest = const_cast<void*>(at(p.rest, p.ot));
  p.lse += start * p.lt;
  p.delta += start * p.lt;
  p.part_k += start * part_pitch(p);
  p.part_v += start * part_pitch(p);
  return (int)(word >> 32);
}

template <class T> __device__ __forceinline__ float ld(const void* p, int64_t i);
template <> __device__ __forceinline__ float ld<float>(const void* p, int64_t i) { return ((const float*)p)[i]; }
template <> __device__ __forceinline__ float ld<bf16_t>(const void* p, int64_t i) {
  return bf16_to_f32(((const bf16_t*)p)[i]);
}
template <class T> __device__ __forceinline__ void st(void* p, int64_t i, float x);
template <> __device__ __forceinline__ void st<float>(void* p, int64_t i, float x) { ((float*)p)[i] = x; }
template <> __device__ __forceinline__ void st<bf16_t>(void* p, int64_t i, float x) {
  ((bf16_t*)p)[i] = f32_to_bf16(x);
}

__device__ __forceinline__ float wave_sum(float x) {
#pragma unroll
  for (int off = 32; off; off >>= 1) x += __shfl_xor(x, off);
  return x;
}

constexpr int GEN_WAVES = 4;  // rows per workgroup

// row -> (b, h, t) and its element offset in a q-shaped array
__device__ __forceinline__ void gen_row(const AttnGenArgs& p, int64_t row, int64_t heads, int64_t& b, int64_t& h,
                                        int64_t& t) {
  t = row % p.time;
  h = (row / p.time) % heads;
  b = row / (p.time * heads);
}

// Output and lse of query t of (b, h).
template <class T, class Args>
__device__ __forceinline__ void fwd_row(const Args& p, int64_t b, int64_t h, int64_t t, int lane) {
  const int64_t kvh = h / (p.heads / p.kv_heads);
  const int64_t qi = b * p.qb + h * p.qh + t * p.qt, kbase = b * p.kb + kvh * p.kh;
  const int64_t oi = b * p.qb + h * p.qh + t * out_pitch(p);
  const int D = (int)p.dim;
  float qv[4], acc[4];
#pragma unroll
  for (int j = 0; j < 4; j++) {
    const int d = lane + 64 * j;
    qv[j] = d < D ? ld<T>(p.q, qi + d) : 0.f;
    acc[j] = 0.f;
  }
  float m = -INFINITY, l = 0.f;
  const int64_t end = p.causal ? t + 1 : p.time;
  for (int64_t s = 0; s < end; s++) {
    const int64_t ki = kbase + s * p.kt, vi = kbase + s * value_pitch(p);
    float dot = 0.f;
#pragma unroll
    for (int j = 0; j < 4; j++) {
      const int d = lane + 64 * j;
      if (d < D) dot += qv[j] * ld<T>(p.k, ki + d);
    }
    const float x = wave_sum(dot) * p.scale;
    const float m_new = fmaxf(m, x);
    const float alpha = __expf(m - m_new), pr = __expf(x - m_new);
    l = l * alpha + pr;
#pragma unroll
    for (int j = 0; j < 4; j++) {
      const int d = lane + 64 * j;
      acc[j] = acc[j] * alpha + (d < D ? pr * ld<T>(p.v, vi + d) : 0.f);
    }
    m = m_new;
  }
  const float inv = l > 0.f ? 1.f / l : 0.f;
#pragma unroll
  for (int j = 0; j < 4; j++) {
    const int d = lane + 64 * j;
    if (d < D) st<T>(p.dq, oi + d, acc[j] * inv);
  }
  if (p.lse && lane == 0) p.lse[b * p.lb + h * p.lh + t * p.lt] = m + __logf(l);
}

// dQ and delta of query t of (b, h).
template <class T, class Args>
__device__ __forceinline__ void bwd_q_row(const Args& p, int64_t b, int64_t h, int64_t t, int lane) {
  const int64_t kvh = h / (p.heads / p.kv_heads);
  const int64_t qi = b * p.qb + h * p.qh + t * p.qt, kbase = b * p.kb + kvh * p.kh;
  const int64_t oi = b * p.qb + h * p.qh + t * out_pitch(p), di = b * p.qb + h * p.qh + t * dq_pitch(p);
  const int64_t li = b * p.lb + h * p.lh + t * p.lt;
  const int D = (int)p.dim;
  float qv[4], gv[4], acc[4], dl = 0.f;
#pragma unroll
  for (int j = 0; j < 4; j++) {
    const int d = lane + 64 * j;
    qv[j] = d < D ? ld<T>(p.q, qi + d) : 0.f;
    gv[j] = d < D ? ld<T>(p.g, oi + d) : 0.f;
    dl += d < D ? gv[j] * ld<T>(p.o, oi + d) : 0.f;
    acc[j] = 0.f;
  }
  dl = wave_sum(dl);
  if (lane == 0) p.delta[li] = dl;
  const float lse = p.lse[li];
  const int64_t end = p.causal ? t + 1 : p.time;
  for (int64_t s = 0; s < end; s++) {
    const int64_t ki = kbase + s * p.kt, vi = kbase + s * value_pitch(p);
    float dot = 0.f, dp = 0.f;
#pragma unroll
    for (int j = 0; j < 4; j++) {
      const int d = lane + 64 * j;
      if (d < D) {
        dot += qv[j] * ld<T>(p.k, ki + d);
        dp += gv[j] * ld<T>(p.v, vi + d);
      }
    }
    const float pr = __expf(wave_sum(dot) * p.scale - lse);
    const float ds = pr * (wave_sum(dp) - dl) * p.scale;
#pragma unroll
    for (int j = 0; j < 4; j++) {
      const int d = lane + 64 * j;
      if (d < D) acc[j] += ds * ld<T>(p.k, ki + d);
    }
  }
#pragma unroll
  for (int j = 0; j < 4; j++) {
    const int d = lane + 64 * j;
    if (d < D) st<T>(p.dq, di + d, acc[j]);
  }
}

// dK and dV of key s of (b, kvh), summed over the query heads [g_lo, g_hi) of
// its group (p.split: head g_lo's unscaled partials).
template <class T, class Args>
__device__ __forceinline__ void bwd_kv_row(const Args& p, int64_t b, int64_t kvh, int64_t s, int lane,
                                           int g_lo, int g_hi) {
  const int64_t head = b * p.kb + kvh * p.kh, ki = head + s * p.kt, vi = head + s * value_pitch(p);
  const int64_t group = p.heads / p.kv_heads;
  const int D = (int)p.dim;
  const float scale = p.split ? 1.f : p.scale;
  float kv_[4], vv[4], ak[4], av[4];
#pragma unroll
  for (int j = 0; j < 4; j++) {
    const int d = lane + 64 * j;
    kv_[j] = d < D ? ld<T>(p.k, ki + d) : 0.f;
    vv[j] = d < D ? ld<T>(p.v, vi + d) : 0.f;
    ak[j] = av[j] = 0.f;
  }
  for (int64_t h = kvh * group + g_lo; h < kvh * group + g_hi; h++) {
    for (int64_t t = p.causal ? s : 0; t < p.time; t++) {
      const int64_t qi = b * p.qb + h * p.qh + t * p.qt;
      const int64_t oi = b * p.qb + h * p.qh + t * out_pitch(p);
      const int64_t li = b * p.lb + h * p.lh + t * p.lt;
      float dot = 0.f, dp = 0.f;
#pragma unroll
      for (int j = 0; j < 4; j++) {
        const int d = lane + 64 * j;
        if (d < D) {
          dot += ld<T>(p.q, qi + d) * kv_[j];
          dp += ld<T>(p.g, oi + d) * vv[j];
        }
      }
      const float pr = __expf(wave_sum(dot) * p.scale - p.lse[li]);
      const float ds = pr * (wave_sum(dp) - p.delta[li]) * scale;
#pragma unroll
      for (int j = 0; j < 4; j++) {
        const int d = lane + 64 * j;
        if (d < D) {
          ak[j] += ds * ld<T>(p.q, qi + d);
          av[j] += pr * ld<T>(p.g, oi + d);
        }
      }
    }
  }
#pragma unroll
  for (int j = 0; j < 4; j++) {
    const int d = lane + 64 * j;
    if (d < D) {
      if (p.split) {
        p.part_k[g_lo * p.part_stride + head + s * part_pitch(p) + d] = ak[j];
        p.part_v[g_lo * p.part_stride + head + s * part_pitch(p) + d] = av[j];
      } else {
        st<T>(p.dk, head + s * dk_pitch(p) + d, ak[j]);
        st<T>(p.dv, head + s * dv_pitch(p) + d, av[j]);
      }
    }
  }
}

template <class T>
__global__ void __launch_bounds__(GEN_WAVES * 64) attention_fwd_rows(AttnGenArgs p) {
  const int64_t row = (int64_t)blockIdx.x * GEN_WAVES + (threadIdx.x >> 6);
  if (row >= p.batch * p.heads * p.time) return;  // whole wave
  int64_t b, h, t;
  gen_row(p, row, p.heads, b, h, t);
  fwd_row<T>(p, b, h, t, threadIdx.x & 63);
}

template <class T>
__global__ void __launch_bounds__(GEN_WAVES * 64) attention_bwd_q_rows(AttnGenArgs p) {
  const int64_t row = (int64_t)blockIdx.x * GEN_WAVES + (threadIdx.x >> 6);
  if (row >= p.batch * p.heads * p.time) return;
  int64_t b, h, t;
  gen_row(p, row, p.heads, b, h, t);
  bwd_q_row<T>(p, b, h, t, threadIdx.x & 63);
}

template <class T>
__global__ void __launch_bounds__(GEN_WAVES * 64) attention_bwd_kv_rows(AttnGenArgs p) {
  const int64_t row = (int64_t)blockIdx.x * GEN_WAVES + (threadIdx.x >> 6);
  if (row >= p.batch * p.kv_heads * p.time) return;
  int64_t b, kvh, s;
  gen_row(p, row, p.kv_heads, b, kvh, s);
  bwd_kv_row<T>(p, b, kvh, s, threadIdx.x & 63, 0, (int)(p.heads / p.kv_heads));
}

}  // namespace
