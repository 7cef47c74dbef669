// RMSNorm of every query and key head and the rotation of its position, in one
// pass: C ABI `qutai_amd_qk_norm_rope`, `_backward`.
//
// A head's row x of D values at position p, with a weight w of D values:
//   r = 1 / sqrt(mean(x^2) + eps),  n = x r w,
//   (y_2i, y_2i+1) = (n_2i, n_2i+1) turned by p theta^(-2i/D)
// and backward, with gn the gradient turned back and t = gn w:
//   dx = r (t - x r^2 mean(t x)),  dw = sum over rows of gn x r.
// Without weights only the turn is left.
//
// An angle is p times its frequency in turns, in 64 bits, less its nearest
// whole number; only the rest, at most half a turn, becomes fp32, which moves the
// sine and cosine by up to pi 2^-24 beside their own rounding (a bf16 result does not
// show it; an fp32 one is off by some three more of its roundings).  Squares, products
// and sums are fp32; a result is rounded once.
//
// Bound by HBM.  32 x 1024 positions of 16 + 4 heads of 64, bf16: forward 34 us
// for 168 MB (4.9 TB/s, a large copy's rate), backward 55 us for 252 MB, weight
// sums 5 us; a wave per row (qk_rows) took 249, 425 and 17.
#include "common.h"
#include "qutai_amd.h"

#include <cmath>
#include <initializer_list>

using namespace qa;

namespace {

constexpr int WAVES = 4;  // of a workgroup

struct QkArgs {
  const void* x[2];   // queries, keys
  const void* g[2];   // their outputs' gradients (backward)
  void* out[2];       // outputs, or input gradients
  const float* w[2];  // null: no norm
  int64_t heads[2], x_row[2], out_row[2];
  const int64_t* starts;  // of each sequence, or null
  int64_t offset, batch, time;
  float* partial;  // backward: [workgroups][2][dim]
  int dim, run;    // run: sequences whose rows of one position are taken together
  int slices;      // waves that share them
  float eps;
  double turns[128];  // frequency of each pair, in turns
};

template <class T> __device__ __forceinline__ float get(const T* p, int64_t i);
template <> __device__ __forceinline__ float get<float>(const float* p, int64_t i) { return p[i]; }
template <> __device__ __forceinline__ float get<bf16_t>(const bf16_t* p, int64_t i) { return bf16_to_f32(p[i]); }
__device__ __forceinline__ void put(float* p, int64_t i, float v) { p[i] = v; }
__device__ __forceinline__ void put(bf16_t* p, int64_t i, float v) { p[i] = f32_to_bf16(v); }

__device__ __forceinline__ int64_t position_of(const QkArgs& a, int64_t b, int64_t t) {
  return a.offset + t + (a.starts ? a.starts[b] : 0);
}

// sine and cosine of position * turns whole turns
__device__ __forceinline__ void turn(int64_t position, double turns, float& s, float& c) {
  const double x = (double)position * turns;
  sincospif(2.f * (float)(x - rint(x)), &s, &c);
}

__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
  for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o);
  return v;
}

// A wave per row, a pair per lane (two for more than 128 values): every width,
// pitch and alignment.
template <class T, bool BACKWARD>
__global__ void __launch_bounds__(WAVES * 64) qk_rows(QkArgs a) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, half = a.dim / 2;
  const int64_t all = a.heads[0] + a.heads[1], rows = a.batch * a.time * all;
  float dw[2][2][2] = {};
  for (int64_t row = blockIdx.x * WAVES + wave; row < rows; row += (int64_t)gridDim.x * WAVES) {
    const int64_t at = row / all, b = at / a.time, t = at % a.time;
    const int64_t hh = row % all;
    const int which = hh < a.heads[0] ? 0 : 1;
    const int64_t h = which ? hh - a.heads[0] : hh;
    const T* x = (const T*)a.x[which] + at * a.x_row[which] + h * a.dim;
    T* out = (T*)a.out[which] + at * a.out_row[which] + h * a.dim;
    const T* g = BACKWARD ? (const T*)a.g[which] + (at * a.heads[which] + h) * a.dim : nullptr;
    const float* w = a.w[which];
    const int64_t position = position_of(a, b, t);
    float v[2][2] = {}, y[2][2] = {}, s[2] = {}, c[2] = {}, squares = 0.f, dots = 0.f;
#pragma unroll
    for (int u = 0; u < 2; u++) {
      const int i = lane + 64 * u;
      if (i >= half) continue;
      turn(position, a.turns[i], s[u], c[u]);
#pragma unroll
      for (int e = 0; e < 2; e++) v[u][e] = get(x, 2 * i + e);
      if constexpr (BACKWARD) {
        const float g0 = get(g, 2 * i), g1 = get(g, 2 * i + 1);
        y[u][0] = fmaf(g0, c[u], g1 * s[u]);
        y[u][1] = fmaf(g1, c[u], -(g0 * s[u]));
      }
      if (w) {
#pragma unroll
        for (int e = 0; e < 2; e++) {
          squares = fmaf(v[u][e], v[u][e], squares);
          if constexpr (BACKWARD) dots = fmaf(y[u][e] * w[2 * i + e], v[u][e], dots);
        }
      }
    }
    float r = 1.f, m = 0.f;
    if (w) {
      r = 1.f / sqrtf(wave_sum(squares) / (float)a.dim + a.eps);
      if constexpr (BACKWARD) m = wave_sum(dots) * r / (float)a.dim;
    }
#pragma unroll
    for (int u = 0; u < 2; u++) {
      const int i = lane + 64 * u;
      if (i >= half) continue;
      const float w0 = w ? w[2 * i] : 1.f, w1 = w ? w[2 * i + 1] : 1.f;
      if constexpr (BACKWARD) {
        const float n0 = v[u][0] * r, n1 = v[u][1] * r;
        dw[which][u][0] = fmaf(y[u][0], n0, dw[which][u][0]);
        dw[which][u][1] = fmaf(y[u][1], n1, dw[which][u][1]);
        put(out, 2 * i, w ? r * fmaf(-n0, m, y[u][0] * w0) : y[u][0]);
        put(out, 2 * i + 1, w ? r * fmaf(-n1, m, y[u][1] * w1) : y[u][1]);
      } else {
        const float n0 = v[u][0] * r * w0, n1 = v[u][1] * r * w1;
        put(out, 2 * i, fmaf(n0, c[u], -(n1 * s[u])));
        put(out, 2 * i + 1, fmaf(n0, s[u], n1 * c[u]));
      }
    }
  }
  if constexpr (BACKWARD) {
    if (!a.partial) return;
    __shared__ float sums[WAVES][2][256];
#pragma unroll
    for (int which = 0; which < 2; which++)
#pragma unroll
      for (int u = 0; u < 2; u++) {
        const int i = lane + 64 * u;
        if (i < half) sums[wave][which][2 * i] = dw[which][u][0], sums[wave][which][2 * i + 1] = dw[which][u][1];
      }
    __syncthreads();
    for (int j = threadIdx.x; j < 2 * a.dim; j += WAVES * 64) {
      const int which = j / a.dim, i = j % a.dim;
      float total = 0.f;
#pragma unroll
      for (int n = 0; n < WAVES; n++) total += sums[n][which][i];
      a.partial[(int64_t)blockIdx.x * 2 * a.dim + j] = total;
    }
  }
}

// The sum over aligned groups of G lanes, in every lane of the group.
template <int CTRL>
__device__ __forceinline__ float dpp(float v) {
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xf, 0xf, true));
}
template <int G>
__device__ __forceinline__ float group_sum(float v) {
  v += dpp<0xB1>(v);                        // lane ^ 1
  v += dpp<0x4E>(v);                        // lane ^ 2
  if constexpr (G >= 8) v += dpp<0x141>(v);   // mirrored in 8: the other four
  if constexpr (G >= 16) v += dpp<0x140>(v);  // mirrored in 16: the other eight
  if constexpr (G >= 32) v += __shfl_xor(v, 16);
  if constexpr (G >= 64) v += __shfl_xor(v, 32);
  return v;
}

template <class T, int E>
__device__ __forceinline__ void unpack(const u32x4& w, float (&v)[E]) {
#pragma unroll
  for (int e = 0; e < E; e++) {
    if constexpr (E == 4) v[e] = __uint_as_float(w[e]);
    else v[e] = __uint_as_float(e & 1 ? w[e >> 1] & 0xffff0000u : w[e >> 1] << 16);
  }
}

// G lanes per row, a 16-byte chunk each, so both values of a pair share a lane; a
// wave takes 64 / G heads of a position at a time, for the same position of `run`
// sequences, whose angles are computed once, with U rows in flight per lane.  Rows
// of whole chunks, 16-byte aligned.
template <class T, int G, bool BACKWARD>
__global__ void __launch_bounds__(WAVES * 64) qk_chunks(QkArgs a) {
  constexpr int E = 16 / (int)sizeof(T), R = 64 / G, U = 4;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = lane % G * E, rr = lane / G;
  const bool in = c < a.dim;
  const float share = 1.f / (float)a.dim;
  float w[2][E], dw[2][E] = {};
#pragma unroll
  for (int side = 0; side < 2; side++)
#pragma unroll
    for (int e = 0; e < E; e++) w[side][e] = a.w[side] && in ? a.w[side][c + e] : 1.f;
  // positions, and those of few positions times their slices, are below 2^31
  const uint32_t runs = (uint32_t)((a.batch + a.run - 1) / a.run), slices = (uint32_t)a.slices;
  const uint32_t items = (uint32_t)a.time * runs * slices;
  for (uint32_t item = uniform32((int)(blockIdx.x * WAVES + wave)); item < items; item += gridDim.x * WAVES) {
    const uint32_t first = item / slices;
    const int64_t t = first / runs, b0 = (int64_t)(first - (uint32_t)t * runs) * a.run;
    int skip = (int)(item - first * slices);  // groups of U rows until this wave's next
    const int n = (int)(a.batch - b0 < a.run ? a.batch - b0 : a.run);
    const int64_t position = position_of(a, b0, t);  // one sequence where they start apart
    float s[E / 2], co[E / 2];
#pragma unroll
    for (int j = 0; j < E / 2; j++) turn(position, in ? a.turns[c / 2 + j] : 0.0, s[j], co[j]);
#pragma unroll
    for (int side = 0; side < 2; side++) {
      const int heads = (int)a.heads[side], turns = (heads + R - 1) / R, jobs = n * turns;
      const bool normed = a.w[side];
      int bb = 0, hi = 0;
      for (int job = 0; job < jobs; job += U) {
        if (skip--) {
          for (hi += U; hi >= turns; hi -= turns) bb++;
          continue;
        }
        skip = a.slices - 1;
        u32x4 x[U], g[U];
        int64_t at[U];
        int head[U];
#pragma unroll
        for (int u = 0; u < U; u++) {
          x[u] = g[u] = u32x4{0u, 0u, 0u, 0u};
          at[u] = (b0 + bb) * a.time + t;
          head[u] = job + u < jobs && in ? hi * R + rr : heads;
          if (++hi == turns) hi = 0, bb++;
          if (head[u] < heads) {
            x[u] = global_load<u32x4>((const T*)a.x[side] + at[u] * a.x_row[side] + head[u] * a.dim + c);
            if constexpr (BACKWARD) g[u] = global_load<u32x4>((const T*)a.g[side] + (at[u] * heads + head[u]) * a.dim + c);
          }
        }
#pragma unroll
        for (int u = 0; u < U; u++) {
          if (job + u >= jobs) break;
          float v[E], y[E];
          unpack<T, E>(x[u], v);
          if constexpr (BACKWARD) {
            float gv[E];
            unpack<T, E>(g[u], gv);
#pragma unroll
            for (int j = 0; j < E / 2; j++) {
              y[2 * j] = fmaf(gv[2 * j], co[j], gv[2 * j + 1] * s[j]);
              y[2 * j + 1] = fmaf(gv[2 * j + 1], co[j], -(gv[2 * j] * s[j]));
            }
          }
          float r = 1.f;
          if (normed) {
            float squares = 0.f;
#pragma unroll
            for (int e = 0; e < E; e++) squares = fmaf(v[e], v[e], squares);
            r = 1.f / sqrtf(fmaf(group_sum<G>(squares), share, a.eps));
#pragma unroll
            for (int e = 0; e < E; e++) v[e] *= r;
            if constexpr (BACKWARD) {
              if (head[u] >= heads)  // no row: nothing for dw, also where eps is 0
#pragma unroll
                for (int e = 0; e < E; e++) v[e] = 0.f;
              float dots = 0.f;
#pragma unroll
              for (int e = 0; e < E; e++) {
                dw[side][e] = fmaf(y[e], v[e], dw[side][e]);
                y[e] *= w[side][e];
                dots = fmaf(y[e], v[e], dots);
              }
              const float m = group_sum<G>(dots) * share;
#pragma unroll
              for (int e = 0; e < E; e++) y[e] = r * fmaf(-v[e], m, y[e]);
            } else {
#pragma unroll
              for (int e = 0; e < E; e++) v[e] *= w[side][e];
            }
          }
          if constexpr (!BACKWARD) {
#pragma unroll
            for (int j = 0; j < E / 2; j++) {
              y[2 * j] = fmaf(v[2 * j], co[j], -(v[2 * j + 1] * s[j]));
              y[2 * j + 1] = fmaf(v[2 * j], s[j], v[2 * j + 1] * co[j]);
            }
          }
          u32x4 o;
#pragma unroll
          for (int e = 0; e < 4; e++) {
            if constexpr (E == 4) o[e] = __float_as_uint(y[e]);
            else o[e] = pack_bf16x2(y[2 * e], y[2 * e + 1]);
          }
          if (head[u] < heads) global_store((T*)a.out[side] + at[u] * a.out_row[side] + head[u] * a.dim + c, o);
        }
      }
    }
  }
  if constexpr (BACKWARD) {
    if (!a.partial) return;
    __shared__ float sums[WAVES][2][256];
#pragma unroll
    for (int side = 0; side < 2; side++)
#pragma unroll
      for (int e = 0; e < E; e++) {
        float v = dw[side][e];
#pragma unroll
        for (int o = G; o < 64; o <<= 1) v += __shfl_xor(v, o);
        if (rr == 0 && in) sums[wave][side][c + e] = v;
      }
    __syncthreads();
    for (int j = threadIdx.x; j < 2 * a.dim; j += WAVES * 64) {
      const int side = j / a.dim, i = j % a.dim;
      float total = 0.f;
#pragma unroll
      for (int n = 0; n < WAVES; n++) total += sums[n][side][i];
      a.partial[(int64_t)blockIdx.x * 2 * a.dim + j] = total;
    }
  }
}

// Weight gradients: the workgroups' sums, added in one order.  A workgroup of
// 1024 threads takes 16 columns of [parts][columns], 64 parts at a time.
__global__ void __launch_bounds__(1024) qk_weights(const float* partial, float* dwq, float* dwk, int parts, int dim) {
  __shared__ float sums[64][17];
  const int column = blockIdx.x * 16 + (threadIdx.x & 15), part = threadIdx.x >> 4, columns = 2 * dim;
  float total = 0.f;
  if (column < columns) {
#pragma unroll 8
    for (int p = part; p < parts; p += 64) total += partial[(int64_t)p * columns + column];
  }
  sums[part][threadIdx.x & 15] = total;
  __syncthreads();
  if (part == 0 && column < columns) {
    total = 0.f;
#pragma unroll
    for (int n = 0; n < 64; n++) total += sums[n][threadIdx.x];
    float* out = column < dim ? dwq : dwk;
    if (out) out[column % dim] = total;
  }
}

constexpr int PARTS = 1024;  // workgroups of the backward, at most

// Whether every row is whole 16-byte chunks.
bool chunked(const QkArgs& a, int es, bool backward) {
  for (int side = 0; side < 2; side++) {
    if (!a.heads[side]) continue;
    if (a.dim * es % 16 || a.x_row[side] * es % 16 || a.out_row[side] * es % 16) return false;
    if ((uintptr_t)a.x[side] % 16 || (uintptr_t)a.out[side] % 16 || (backward && (uintptr_t)a.g[side] % 16)) return false;
  }
  return true;
}

// Sequences whose rows of a position share their angles: as many as leave
// `waves` waves, where all start together.  Fewer positions than that are shared
// out over several waves each, by groups of four rows per lane.
int64_t set_run(QkArgs& a, int64_t waves, int es) {
  const int64_t run = a.starts ? 1 : a.batch * a.time / waves;
  a.run = (int)(run < 1 ? 1 : run > a.batch ? a.batch : run > 64 ? 64 : run);
  const int64_t items = a.time * ((a.batch + a.run - 1) / a.run);
  int lanes = 4, groups = 0;
  while (lanes * 16 / es < a.dim) lanes *= 2;
  for (const int64_t heads : a.heads) groups += (int)(((heads * lanes + 63) / 64 * a.run + 3) / 4);
  const int64_t slices = items < waves ? (waves + items - 1) / items : 1;
  a.slices = (int)(slices < groups ? slices : groups);
  return items * a.slices;
}

// The number of workgroups launched.
template <class T, bool BACKWARD>
int launch(QkArgs& a, hipStream_t stream) {
  const int64_t most = BACKWARD ? PARTS : 1 << 20;
  const bool chunks = chunked(a, sizeof(T), BACKWARD);
  int64_t items = a.batch * a.time * (a.heads[0] + a.heads[1]);
  if (chunks) items = set_run(a, BACKWARD ? PARTS * WAVES : 8192, sizeof(T));
  const int64_t blocks = (items + WAVES - 1) / WAVES < most ? (items + WAVES - 1) / WAVES : most;
  const dim3 grid((unsigned)blocks), block(WAVES * 64);
  const int lanes = a.dim * (int)sizeof(T) / 16;
  if (!chunks) hipLaunchKernelGGL((qk_rows<T, BACKWARD>), grid, block, 0, stream, a);
  else if (lanes <= 4) hipLaunchKernelGGL((qk_chunks<T, 4, BACKWARD>), grid, block, 0, stream, a);
  else if (lanes <= 8) hipLaunchKernelGGL((qk_chunks<T, 8, BACKWARD>), grid, block, 0, stream, a);
  else if (lanes <= 16) hipLaunchKernelGGL((qk_chunks<T, 16, BACKWARD>), grid, block, 0, stream, a);
  else if (lanes <= 32) hipLaunchKernelGGL((qk_chunks<T, 32, BACKWARD>), grid, block, 0, stream, a);
  else if constexpr (sizeof(T) == 4) hipLaunchKernelGGL((qk_chunks<T, 64, BACKWARD>), grid, block, 0, stream, a);
  return (int)blocks;
}

int fill_args(QkArgs& a, const void* q, const void* k, const float* wq, const float* wk, void* q_out, void* k_out,
              const int64_t* starts, int64_t offset, int64_t batch, int64_t time, int64_t heads, int64_t kv_heads,
              int64_t dim, int64_t q_row, int64_t k_row, int64_t q_out_row, int64_t k_out_row, double theta, double eps,
              int dtype) {
  if (batch < 0 || time < 0 || heads < 0 || kv_heads < 0 || heads + kv_heads == 0) return QA_EINVAL;
  if (dim <= 0 || dim % 2 || dim > 256 || (dtype != BF16 && dtype != F32)) return QA_EINVAL;
  if (heads > (1 << 20) || kv_heads > (1 << 20) || q_row < heads * dim || k_row < kv_heads * dim) return QA_EINVAL;
  if (q_out_row < heads * dim || k_out_row < kv_heads * dim) return QA_EINVAL;
  const int64_t most = 1ll << 40;
  if (q_row > most || k_row > most || q_out_row > most || k_out_row > most) return QA_EINVAL;
  if (time && batch > 0x7fffffff / time) return QA_EINVAL;
  for (const int64_t row : {q_row, k_row, q_out_row, k_out_row})
    if (row && batch * time > (1ll << 60) / row) return QA_EINVAL;
  if (!(theta > 0.0) || theta > 1e30 || !(eps >= 0.0) || eps > 1e30) return QA_EINVAL;
  if (offset > most || offset < -most) return QA_EINVAL;
  if (batch * time) {
    if (heads && (!q || !q_out)) return QA_EINVAL;
    if (kv_heads && (!k || !k_out)) return QA_EINVAL;
  }
  if (heads && kv_heads && !wq != !wk) return QA_EINVAL;  // both are normed or neither is
  a.x[0] = q, a.x[1] = k, a.out[0] = q_out, a.out[1] = k_out, a.w[0] = wq, a.w[1] = wk;
  a.g[0] = a.g[1] = nullptr;
  a.heads[0] = heads, a.heads[1] = kv_heads;
  a.x_row[0] = q_row, a.x_row[1] = k_row, a.out_row[0] = q_out_row, a.out_row[1] = k_out_row;
  a.starts = starts, a.offset = offset, a.batch = batch, a.time = time, a.run = a.slices = 1, a.partial = nullptr;
  a.dim = (int)dim, a.eps = (float)eps;
  const double whole = 6.283185307179586476925287;
  for (int i = 0; i < dim / 2; i++) a.turns[i] = std::pow(theta, -2.0 * i / (double)dim) / whole;
  return QA_OK;
}

}  // namespace

extern "C" int qutai_amd_qk_norm_rope(const void* q, const void* k, const float* q_weight, const float* k_weight,
                                      void* q_out, void* k_out, const int64_t* starts, int64_t offset, int64_t batch,
                                      int64_t time, int64_t heads, int64_t kv_heads, int64_t dim, int64_t q_row,
                                      int64_t k_row, double theta, double eps, int dtype, void* stream_) {
  QkArgs a;
  const int status = fill_args(a, q, k, q_weight, k_weight, q_out, k_out, starts, offset, batch, time, heads, kv_heads,
                               dim, q_row, k_row, heads * dim, kv_heads * dim, theta, eps, dtype);
  if (status) return status;
  if (batch * time == 0) return QA_OK;
  hipStream_t stream = (hipStream_t)stream_;
  if (dtype == BF16) launch<bf16_t, false>(a, stream);
  else launch<float, false>(a, stream);
  return (int)hipGetLastError();
}

extern "C" int64_t qutai_amd_qk_norm_rope_workspace(int64_t dim) {
  return dim > 0 && dim <= 256 ? (int64_t)PARTS * 2 * dim : 0;
}

extern "C" int qutai_amd_qk_norm_rope_backward(const void* gq, const void* gk, const void* q, const void* k,
                                               const float* q_weight, const float* k_weight, void* dq, void* dk,
                                               float* dq_weight, float* dk_weight, const int64_t* starts,
                                               int64_t offset, int64_t batch, int64_t time, int64_t heads,
                                               int64_t kv_heads, int64_t dim, int64_t q_row, int64_t k_row,
                                               int64_t dq_row, int64_t dk_row, double theta, double eps, int dtype,
                                               float* workspace, int64_t workspace_floats, void* stream_) {
  QkArgs a;
  const int status = fill_args(a, q, k, q_weight, k_weight, dq, dk, starts, offset, batch, time, heads, kv_heads, dim,
                               q_row, k_row, dq_row, dk_row, theta, eps, dtype);
  if (status) return status;
  if (batch * time && ((heads && !gq) || (kv_heads && !gk))) return QA_EINVAL;
  const bool weights = dq_weight || dk_weight;
  if ((dq_weight && !q_weight) || (dk_weight && !k_weight)) return QA_EINVAL;
  if (weights && (!workspace || workspace_floats < (int64_t)PARTS * 2 * dim)) return QA_EWORKSPACE;
  a.g[0] = gq, a.g[1] = gk, a.partial = weights ? workspace : nullptr;
  hipStream_t stream = (hipStream_t)stream_;
  int parts = 0;
  if (batch * time) parts = dtype == BF16 ? launch<bf16_t, true>(a, stream) : launch<float, true>(a, stream);
  if (weights)
    hipLaunchKernelGGL(qk_weights, dim3((unsigned)((2 * dim + 15) / 16)), dim3(1024), 0, stream, workspace, dq_weight,
                       dk_weight, parts, (int)dim);
  return (int)hipGetLastError();
}
