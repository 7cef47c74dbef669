// Rotary positions of query and key heads: C ABI `qutai_amd_rotary`, and the places of
// packed sequences' tokens: `qutai_amd_positions`.
//
// Pair i of a head's first R channels is turned by its token's position p times
// turns[i] whole turns and scaled by `magnitude`:
//   (a, b) -> magnitude (a cos - b sin, a sin + b cos),
// with (a, b) channels (2i, 2i + 1), or (i, i + R/2) in the half layout; channels
// from R on are copied.  The inverse turns back by the same angle (it is the
// gradient: the transpose of the turn and its magnitude).
//
// An angle is p times its frequency in 64 bits, less its nearest whole number of
// turns; the rest becomes fp32 and what that rounding leaves, which corrects sine
// and cosine to first order, so positions far beyond 2^24 / 2 pi keep fp32's bits.
//
// A lane takes V pairs (16 bytes of either half) of one token, computes their
// angles once and turns them in every SLOTS-th head of queries and keys.  Memory bounds
// it: 32768 tokens, 32 and 8 bf16 heads of 128 from the columns of a product, 133 us for
// 671 MB (5.0 TB/s, a copy 4.9); 1001 tokens, 12 and 12 fp32 heads of 80, 6.5 us for 15 MB,
// of which 5 are a launch's and the angles' (8 tokens take as long).
#include "common.h"
#include "qutai_amd.h"

#include <algorithm>

using namespace qa;

namespace {

constexpr int THREADS = 256;

struct RotaryArgs {
  const void* x[2];  // queries, keys
  void* out[2];
  int64_t x_row[2], out_row[2];
  const int64_t* positions;  // of every token, or null: offset + starts[b] + t
  const int64_t* starts;
  int64_t offset, tokens, time;
  int heads[2], dim, rotary;
  int pair_lanes, lanes, slots;  // lanes of a token that turn pairs, all of its lanes, lanes that share its heads
  float magnitude, sign;
  double turns[128];
};

// N elements at once: 16 or 8 bytes, or one.  Inputs are read once, past the caches;
// results stay there for the attention that reads them next (336 MB of them, more than the
// caches hold, take 133 us either way).
template <class T, int N>
__device__ __forceinline__ void load(const T* p, float (&v)[N]) {
  if constexpr (N == 1) {
    if constexpr (sizeof(T) == 4) v[0] = p[0];
    else v[0] = bf16_to_f32(p[0]);
  } else {
    typedef uint32_t words __attribute__((__vector_size__(sizeof(T) * N)));
    const words w = global_load_nt<words>(p);
#pragma unroll
    for (int e = 0; e < N; e++) {
      if constexpr (sizeof(T) == 4) v[e] = __uint_as_float(w[e]);
      else v[e] = __uint_as_float(e & 1 ? w[e / 2] & 0xffff0000u : w[e / 2] << 16);
    }
  }
}
template <class T, int N>
__device__ __forceinline__ void store(T* p, const float (&v)[N]) {
  if constexpr (N == 1) {
    if constexpr (sizeof(T) == 4) p[0] = v[0];
    else p[0] = f32_to_bf16(v[0]);
  } else {
    typedef uint32_t words __attribute__((__vector_size__(sizeof(T) * N)));
    words w;
#pragma unroll
    for (int e = 0; e < (int)(sizeof(T) * N / 4); e++) {
      if constexpr (sizeof(T) == 4) w[e] = __float_as_uint(v[e]);
      else w[e] = pack_bf16x2(v[2 * e], v[2 * e + 1]);
    }
    global_store(p, w);
  }
}

// V elements of T at a time: 16 or 8 bytes, or one where widths, pitches or addresses
// are no whole chunks of that (32768 tokens, 16 and 4 bf16 heads of 80: 54 us with 32
// channels turned, 124 with 20, whose halves of 10 are 20 bytes).
template <class T, int V, bool HALF>
__global__ void __launch_bounds__(THREADS) rotary_kernel(RotaryArgs a) {
  const int64_t id = (int64_t)blockIdx.x * THREADS + threadIdx.x;
  const int lane = (int)(id % a.lanes);
  const int64_t rest = id / a.lanes;
  const int slot = (int)(rest % a.slots);
  const int64_t token = rest / a.slots;
  if (token >= a.tokens) return;
  const bool turned = lane < a.pair_lanes;
  // the two chunks of the lane: the halves of its pairs, or (interleaved) V pairs
  // side by side, or two chunks that are copied
  const int tail = a.rotary + 2 * V * (lane - a.pair_lanes);
  const int first = !turned ? tail : HALF ? V * lane : 2 * V * lane;
  const int second = turned && HALF ? first + a.rotary / 2 : first + V;
  const bool both = turned || second < a.dim;
  float c[V], s[V];
  if (turned) {
    const int64_t at = a.positions ? a.positions[token]
                                   : a.offset + token % a.time + (a.starts ? a.starts[token / a.time] : 0);
#pragma unroll
    for (int e = 0; e < V; e++) {
      const double turns = (double)at * a.turns[V * lane + e], left = turns - rint(turns);
      const float near = (float)left, off = 6.2831855f * (float)(left - (double)near);
      float sn, cs;
      sincospif(2.f * near, &sn, &cs);
      c[e] = fmaf(-sn, off, cs) * a.magnitude;
      s[e] = fmaf(cs, off, sn) * a.magnitude * a.sign;
    }
  }
  for (int h = slot; h < a.heads[0] + a.heads[1]; h += a.slots) {
    const int side = h >= a.heads[0];
    const int64_t head = (int64_t)(side ? h - a.heads[0] : h) * a.dim;
    const T* x = (const T*)a.x[side] + token * a.x_row[side] + head;
    T* out = (T*)a.out[side] + token * a.out_row[side] + head;
    float u[V], w[V];
    load<T, V>(x + first, u);
    if (both) load<T, V>(x + second, w);
    if (turned) {
      if constexpr (HALF) {
#pragma unroll
        for (int e = 0; e < V; e++) {
          const float p = u[e], q = w[e];
          u[e] = fmaf(p, c[e], -(q * s[e]));
          w[e] = fmaf(q, c[e], p * s[e]);
        }
      } else {
        float y[2 * V];
#pragma unroll
        for (int e = 0; e < V; e++) y[e] = u[e], y[V + e] = w[e];
#pragma unroll
        for (int e = 0; e < V; e++) {
          const float p = y[2 * e], q = y[2 * e + 1];
          y[2 * e] = fmaf(p, c[e], -(q * s[e]));
          y[2 * e + 1] = fmaf(q, c[e], p * s[e]);
        }
#pragma unroll
        for (int e = 0; e < V; e++) u[e] = y[e], w[e] = y[V + e];
      }
    }
    store<T, V>(out + first, u);
    if (both) store<T, V>(out + second, w);
  }
}

template <class T, int V>
hipError_t launch(RotaryArgs& a, bool half, hipStream_t stream) {
  a.pair_lanes = a.rotary / (2 * V);
  a.lanes = a.pair_lanes + (a.dim - a.rotary + 2 * V - 1) / (2 * V);
  a.slots = std::max(1, std::min(8, (a.heads[0] + a.heads[1] + 3) / 4));
  const int64_t threads = a.tokens * a.slots * a.lanes;
  if (threads > 0xffffff00ll) return hipErrorInvalidValue;
  const dim3 grid((unsigned)((threads + THREADS - 1) / THREADS));
  if (half) hipLaunchKernelGGL((rotary_kernel<T, V, true>), grid, dim3(THREADS), 0, stream, a);
  else hipLaunchKernelGGL((rotary_kernel<T, V, false>), grid, dim3(THREADS), 0, stream, a);
  return hipGetLastError();
}

// A token's place in its sequence, found among the sequences' starts by halving; 0
// behind the last one.
__global__ void __launch_bounds__(THREADS) positions_kernel(const int64_t* starts, int64_t sequences, int64_t used,
                                                            int64_t total, int64_t* positions) {
  const int64_t t = (int64_t)blockIdx.x * THREADS + threadIdx.x;
  if (t >= total) return;
  int64_t lo = 0, hi = sequences;
  while (hi - lo > 1) {
    const int64_t mid = (lo + hi) >> 1;
    if (starts[mid] <= t) lo = mid;
    else hi = mid;
  }
  positions[t] = t < used ? t - starts[lo] : 0;
}

}  // namespace

extern "C" {

int qutai_amd_positions(const int64_t* starts, int64_t sequences, int64_t used, int64_t total, int64_t* positions,
                        void* stream) {
  if (sequences < 0 || used < 0 || used > total || total >= 1ll << 31 || (used && !sequences)) return QA_EINVAL;
  if (!total) return QA_OK;
  if (!positions || (used && !starts)) return QA_EINVAL;
  const unsigned grid = (unsigned)((total + THREADS - 1) / THREADS);
  hipLaunchKernelGGL(positions_kernel, dim3(grid), dim3(THREADS), 0, (hipStream_t)stream, starts, used ? sequences : 0, used,
                     total, positions);
  return (int)hipGetLastError();
}

int qutai_amd_rotary(const void* q, const void* k, void* q_out, void* k_out, const double* turns, const int64_t* positions,
                     const int64_t* starts, int64_t offset, int64_t batch, int64_t time, int64_t heads, int64_t kv_heads,
                     int64_t dim, int64_t rotary, int64_t q_row, int64_t k_row, int64_t q_out_row, int64_t k_out_row, int half,
                     double magnitude, int inverse, int dtype, void* stream) {
  const int64_t most = 1 << 20;
  if (batch < 0 || time < 0 || heads < 0 || kv_heads < 0 || heads > most || kv_heads > most || heads + kv_heads == 0)
    return QA_EINVAL;
  if (dim <= 0 || dim > 256 || rotary < 0 || rotary > dim || rotary % 2 || (rotary && !turns)) return QA_EINVAL;
  if ((dtype != F32 && dtype != BF16) || !(magnitude > 0.0) || !(magnitude < 1e30)) return QA_EINVAL;
  if (time && batch > 0x7fffffff / time) return QA_EINVAL;
  RotaryArgs a = {};
  const int64_t n[2] = {heads, kv_heads}, rows[2] = {q_row, k_row}, out_rows[2] = {q_out_row, k_out_row};
  const void* x[2] = {q, k};
  void* out[2] = {q_out, k_out};
  const int64_t item = dtype == F32 ? 4 : 2;
  int64_t odd = 0;  // what has to be whole chunks, or'd
  for (int i = 0; i < 2; i++) {
    if (!n[i]) continue;
    if (rows[i] < n[i] * dim || out_rows[i] < n[i] * dim || rows[i] > (1ll << 40) || out_rows[i] > (1ll << 40))
      return QA_EINVAL;
    if (batch * time && (!x[i] || !out[i])) return QA_EINVAL;
    odd |= (int64_t)(uintptr_t)x[i] | (int64_t)(uintptr_t)out[i] | rows[i] * item | out_rows[i] * item;
    a.x[i] = x[i];
    a.out[i] = out[i];
    a.x_row[i] = rows[i];
    a.out_row[i] = out_rows[i];
    a.heads[i] = (int)n[i];
  }
  if (batch * time == 0) return QA_OK;
  a.positions = positions;
  a.starts = starts;
  a.offset = offset;
  a.tokens = batch * time;
  a.time = time;
  a.dim = (int)dim;
  a.rotary = (int)rotary;
  a.magnitude = (float)magnitude;
  a.sign = inverse ? -1.f : 1.f;
  for (int64_t i = 0; i < rotary / 2; i++) a.turns[i] = turns[i];
  const hipStream_t s = (hipStream_t)stream;
  hipError_t e;
  odd |= rotary / 2 * item | dim * item;
  if (dtype == F32) {
    if (odd % 16 == 0) e = launch<float, 4>(a, half, s);
    else if (odd % 8 == 0) e = launch<float, 2>(a, half, s);
    else e = launch<float, 1>(a, half, s);
  } else {
    if (odd % 16 == 0) e = launch<bf16_t, 8>(a, half, s);
    else if (odd % 8 == 0) e = launch<bf16_t, 4>(a, half, s);
    else e = launch<bf16_t, 1>(a, half, s);
  }
  return e == hipErrorInvalidValue ? QA_EINVAL : (int)e;
}

}  // extern "C"
