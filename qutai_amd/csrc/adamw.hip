// One AdamW step over many tensors: C ABI `qutai_amd_adamw`, `_norm`, `_moments`.
//
//   g' = g min(1, max_norm / norm)
//   m' = b1 m + (1 - b1) g',  v' = b2 v + (1 - b2) g'^2
//   p' = p (1 - lr decay) - (lr / c1) m' / (sqrt(v') / sqrt(c2) + eps),
// c1 = 1 - b1^t and c2 = 1 - b2^t computed by the caller's step number in 64
// bits.  Moments are held in fp32, or in 8 bits:
//
// A block of 256 values of a tensor has an exponent E per moment: the largest
// magnitude's, one more where that is at least 1.875 2^E (so that no code
// overflows), -64 at the least.  Magnitude codes are small floating point numbers
// with three fraction bits, whose top binade is [2^E, 2^(E+1)): the first moment a
// sign and 15 binades, the second 31 binades; code 8 j + f stands for (8 + f) 2^(L
// + j - 4), j > 0, and f 2^(L - 3), j = 0, L the lowest binade's exponent.  A value
// is rounded up with the chance of its nearness to the upper code (16 bits of a
// hash of seed, step, tensor and element), so that the average of moments whose
// change in one step is far below a code's follows them: rounded to nearest, b2 =
// 0.999 would never let a second moment fall.  A positive second moment keeps the
// least code, so a step is never divided by a root that rounding made 0.  Moments
// of 8 bits are computed in 64 (memory bounds the step all the same), so that the
// codes are those of the definition whatever the order of operations.
//
// A block with an infinity or NaN has the exponent 127 and reads as NaN.
#include "common.h"
#include "qutai_amd.h"

#include <algorithm>

using namespace qa;

namespace {

constexpr int THREADS = 256, BLOCK = 256;     // BLOCK: values that share an exponent
constexpr int CHUNK = 4096;                   // values of a workgroup's turn
constexpr int TENSORS = 48;                   // of a launch: their records fit the kernel's arguments
constexpr int NORM_GROUPS = 1024;             // partial sums of a launch
constexpr int NOT_FINITE = 127;

struct Tensor {
  void* p;
  const void* g;
  void* m;
  void* v;
  int8_t* e;
  int64_t count;
  uint32_t chunks;  // of the tensors before it in this launch
  uint32_t key;     // of its rounding
  int bf16, whole;  // whole: 16-byte aligned
};

struct StepArgs {
  int n;
  uint32_t chunks;
  double b1, b1_rest, b2, b2_rest;
  float keep, rate, root, eps;  // 1 - lr decay, lr / c1, 1 / sqrt(c2)
  const double* partial;        // sums of squares, or null
  int partials;
  double max_norm;
  double* norm;
  Tensor t[TENSORS];
};

struct NormArgs {
  int n;
  uint32_t chunks;
  double* partial;
  Tensor t[TENSORS];
};

// The record that holds chunk c.
template <class Args>
__device__ __forceinline__ int tensor_of(const Args& a, uint32_t c) {
  int lo = 0, hi = a.n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (a.t[mid].chunks <= c) lo = mid;
    else hi = mid;
  }
  return lo;
}

__device__ __forceinline__ float get(const void* x, int64_t i, int bf16) {
  return bf16 ? bf16_to_f32(((const bf16_t*)x)[i]) : ((const float*)x)[i];
}
__device__ __forceinline__ void put(void* x, int64_t i, float v, int bf16) {
  if (bf16) ((bf16_t*)x)[i] = f32_to_bf16(v);
  else ((float*)x)[i] = v;
}

// Sum over a workgroup, the same in every thread; the order is fixed.
__device__ __forceinline__ double group_sum(double x, double* shared) {
#pragma unroll
  for (int o = 32; o; o >>= 1) x += __shfl_xor(x, o);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) shared[threadIdx.x >> 6] = x;
  __syncthreads();
  return (shared[0] + shared[1]) + (shared[2] + shared[3]);
}

__global__ void __launch_bounds__(THREADS) adamw_norm(NormArgs a) {
  __shared__ double shared[4];
  double sum = 0.0;
  for (uint32_t c = blockIdx.x; c < a.chunks; c += gridDim.x) {
    const Tensor& t = a.t[tensor_of(a, c)];
    const int64_t start = (int64_t)(c - t.chunks) * CHUNK, end = min(t.count, start + CHUNK);
    for (int64_t i = start + threadIdx.x; i < end; i += THREADS) {
      const double g = get(t.g, i, t.bf16);
      sum += g * g;
    }
  }
  sum = group_sum(sum, shared);
  if (threadIdx.x == 0) a.partial[blockIdx.x] = sum;
}

__device__ __forceinline__ uint32_t mixed(uint32_t x) {
  x ^= x >> 15;
  x *= 0xBB67AE85u;
  x ^= x >> 13;
  x *= 0x6A09E667u;
  return x ^ (x >> 16);
}

__device__ __forceinline__ float decoded(uint32_t code, int least) {
  const int above = max((int)(code >> 3), 1) - 1;
  return ldexpf((float)((int)code - 8 * above), least + above - 3);
}

__device__ __forceinline__ uint32_t high_word(double x) { return (uint32_t)((uint64_t)__double_as_longlong(x) >> 32); }

// The exponent of a block from the largest high word of its values' magnitudes.
__device__ __forceinline__ int block_exponent(uint32_t most) {
  if (most >= 0x7ff00000u) return NOT_FINITE;
  const int e = (int)(most >> 20) - 1023 + ((most >> 17 & 7) == 7);
  return e > NOT_FINITE - 1 ? NOT_FINITE : e < -64 ? -64 : e;
}

__device__ __forceinline__ uint32_t coded(double magnitude, int least, uint32_t bits) {
  const int mine = max((int)(high_word(magnitude) >> 20) - 1023, least);
  return (uint32_t)(mine - least) * 8 + (uint32_t)(ldexp(magnitude, 3 - mine) + (double)bits * 0x1p-16);
}

__device__ __forceinline__ uint32_t wave_max(uint32_t x) {
#pragma unroll
  for (int o = 32; o; o >>= 1) x = max(x, (uint32_t)__shfl_xor((int)x, o));
  return x;
}

template <bool EIGHT>
__global__ void __launch_bounds__(THREADS) adamw_step(StepArgs a) {
#pragma clang fp contract(off)
  __shared__ double shared[4];
  double factor = 1.0;
  if (a.partial) {
    double sum = 0.0;
    for (int i = threadIdx.x; i < a.partials; i += THREADS) sum += a.partial[i];
    const double norm = sqrt(group_sum(sum, shared));
    if (a.norm && blockIdx.x == 0 && threadIdx.x == 0) *a.norm = norm;
    if (!(norm < INFINITY)) return;  // the whole step is left out
    factor = norm > a.max_norm ? a.max_norm / norm : 1.0;
  }
  for (uint32_t c = blockIdx.x; c < a.chunks; c += gridDim.x) {
    const Tensor& t = a.t[tensor_of(a, c)];
    const int64_t start = (int64_t)(c - t.chunks) * CHUNK, end = min(t.count, start + CHUNK);
    if constexpr (EIGHT) {
      const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
      for (int64_t base = start + wave * BLOCK; base < end; base += 4 * BLOCK) {
        int8_t* e = t.e + base / BLOCK * 2;
        const int e1 = e[0], e2 = e[1];
        double m[4], v[4];
        uint32_t most1 = 0, most2 = 0;
#pragma unroll
        for (int j = 0; j < 4; j++) {
          const int64_t i = base + lane * 4 + j;
          m[j] = v[j] = 0.0;
          if (i >= end) continue;
          const uint32_t c1 = ((const uint8_t*)t.m)[i], c2 = ((const uint8_t*)t.v)[i];
          float m0 = decoded(c1 & 127, e1 - 14), v0 = decoded(c2, e2 - 30);
          if (c1 & 128) m0 = -m0;
          if (e1 == NOT_FINITE) m0 = NAN;
          if (e2 == NOT_FINITE) v0 = NAN;
          const double g = (double)get(t.g, i, t.bf16) * factor;
          m[j] = a.b1 * (double)m0 + a.b1_rest * g;
          v[j] = a.b2 * (double)v0 + a.b2_rest * (g * g);
          most1 = max(most1, high_word(m[j]) & 0x7fffffffu);
          most2 = max(most2, high_word(v[j]) & 0x7fffffffu);
        }
        const int E1 = block_exponent(wave_max(most1)), E2 = block_exponent(wave_max(most2));
#pragma unroll
        for (int j = 0; j < 4; j++) {
          const int64_t i = base + lane * 4 + j;
          if (i >= end) continue;
          const uint32_t bits = mixed((uint32_t)i * 0x9E3779B9u + t.key);
          uint32_t c1 = 0, c2 = 0;
          if (E1 != NOT_FINITE) c1 = coded(fabs(m[j]), E1 - 14, bits & 0xffff) | (m[j] < 0.0 ? 128 : 0);
          if (E2 != NOT_FINITE) {
            c2 = coded(v[j], E2 - 30, bits >> 16);
            if (c2 == 0 && v[j] > 0.0) c2 = 1;
          }
          ((uint8_t*)t.m)[i] = (uint8_t)c1;
          ((uint8_t*)t.v)[i] = (uint8_t)c2;
          const float p = get(t.p, i, t.bf16);
          const float step = (float)m[j] / (sqrtf((float)v[j]) * a.root + a.eps);
          put(t.p, i, p * a.keep - a.rate * step, t.bf16);
        }
        if (lane == 0) e[0] = (int8_t)E1, e[1] = (int8_t)E2;
      }
    } else {
      const float f = (float)factor, b1 = (float)a.b1, r1 = (float)a.b1_rest, b2 = (float)a.b2, r2 = (float)a.b2_rest;
      for (int64_t i = start + threadIdx.x; i < end; i += THREADS) {
        const float g = get(t.g, i, t.bf16) * f, p = get(t.p, i, t.bf16);
        const float m = b1 * ((const float*)t.m)[i] + r1 * g, v = b2 * ((const float*)t.v)[i] + r2 * (g * g);
        ((float*)t.m)[i] = m;
        ((float*)t.v)[i] = v;
        put(t.p, i, p * a.keep - a.rate * (m / (sqrtf(v) * a.root + a.eps)), t.bf16);
      }
    }
  }
}

__global__ void __launch_bounds__(THREADS) adamw_moments(const uint8_t* m, const uint8_t* v, const int8_t* e, float* first,
                                                         float* second, int64_t count) {
  for (int64_t i = (int64_t)blockIdx.x * THREADS + threadIdx.x; i < count; i += (int64_t)gridDim.x * THREADS) {
    const int e1 = e[i / BLOCK * 2], e2 = e[i / BLOCK * 2 + 1];
    const float x = decoded(m[i] & 127, e1 - 14);
    first[i] = e1 == NOT_FINITE ? NAN : m[i] & 128 ? -x : x;
    second[i] = e2 == NOT_FINITE ? NAN : decoded(v[i], e2 - 30);
  }
}

// Records of up to TENSORS tensors from `first` on; returns how many tensors
// they took (those without values among them), or a negative status.
template <class Args>
int64_t take(Args& a, const int64_t* tensors, int64_t first, int64_t count, int bits, uint32_t key, bool gradients_only) {
  a.n = 0;
  a.chunks = 0;
  int64_t i = first;
  for (; i < count && a.n < TENSORS; i++) {
    const int64_t* r = tensors + 8 * i;
    const int64_t values = r[5];
    if (values == 0) continue;
    const int64_t chunks = (values + CHUNK - 1) / CHUNK;
    if (a.chunks + chunks > 0x7fffffff) break;
    Tensor& t = a.t[a.n++];
    t.p = (void*)r[0];
    t.g = (const void*)r[1];
    t.m = (void*)r[2];
    t.v = (void*)r[3];
    t.e = (int8_t*)r[4];
    t.count = values;
    t.chunks = a.chunks;
    t.bf16 = r[6] == BF16;
    t.whole = (r[0] | r[1] | r[2] | r[3]) % 16 == 0;
    uint32_t x = key + (uint32_t)r[7];
    x ^= x >> 15;
    x *= 0xBB67AE85u;
    x ^= x >> 13;
    x *= 0x6A09E667u;
    t.key = x ^ (x >> 16);
    a.chunks += (uint32_t)chunks;
  }
  return i - first;
}

uint32_t host_mixed(uint32_t x) {
  x ^= x >> 15;
  x *= 0xBB67AE85u;
  x ^= x >> 13;
  x *= 0x6A09E667u;
  return x ^ (x >> 16);
}

int64_t launches(const int64_t* tensors, int64_t count) {
  int64_t n = 0, chunks = 0, launched = 0;
  for (int64_t i = 0; i < count; i++) {
    const int64_t values = tensors[8 * i + 5], c = (values + CHUNK - 1) / CHUNK;
    if (values == 0) continue;
    if (n == TENSORS || chunks + c > 0x7fffffff) launched++, n = 0, chunks = 0;
    n++;
    chunks += c;
  }
  return launched + (n > 0);
}

bool valid(const int64_t* tensors, int64_t count, int bits, bool gradients_only) {
  if (count < 0 || (count && !tensors)) return false;
  for (int64_t i = 0; i < count; i++) {
    const int64_t* r = tensors + 8 * i;
    if (r[5] < 0 || r[5] > (1ll << 42) || (r[6] != F32 && r[6] != BF16)) return false;
    if (r[5] == 0) continue;
    if (!r[1] || r[1] % (r[6] == BF16 ? 2 : 4)) return false;
    if (gradients_only) continue;
    if (!r[0] || r[0] % (r[6] == BF16 ? 2 : 4) || !r[2] || !r[3]) return false;
    if (bits == 8 ? !r[4] : r[2] % 4 || r[3] % 4) return false;
  }
  return true;
}

}  // namespace

extern "C" {

int64_t qutai_amd_adamw_workspace(const int64_t* tensors, int64_t count) {
  return valid(tensors, count, 32, true) ? launches(tensors, count) * NORM_GROUPS : 0;
}

int qutai_amd_adamw(const int64_t* tensors, int64_t count, int bits, double rate, double beta1, double beta2,
                    double eps, double weight_decay, int64_t step, uint64_t seed, double max_norm, double* workspace,
                    int64_t workspace_values, double* norm, void* stream) {
  if ((bits != 8 && bits != 32) || !valid(tensors, count, bits, false)) return QA_EINVAL;
  if (!(beta1 >= 0.0 && beta1 < 1.0 && beta2 >= 0.0 && beta2 < 1.0) || !(eps > 0.0) || step < 1) return QA_EINVAL;
  if (!(rate >= 0.0) || !(rate < 1e30) || !(weight_decay >= 0.0) || !(weight_decay < 1e30) || !(max_norm >= 0.0))
    return QA_EINVAL;
  const int64_t parts = launches(tensors, count) * NORM_GROUPS;
  if (max_norm > 0.0 && parts && (!workspace || (uintptr_t)workspace % 8 || workspace_values < parts)) return QA_EWORKSPACE;
  if (max_norm > 0.0 && parts) {
    NormArgs a = {};
    int64_t at = 0;
    for (int64_t first = 0; first < count;) {
      first += take(a, tensors, first, count, bits, 0, true);
      if (!a.n) continue;
      a.partial = workspace + at * NORM_GROUPS;
      at++;
      // every partial sum is written: workgroups without a chunk write 0
      hipLaunchKernelGGL(adamw_norm, dim3(NORM_GROUPS), dim3(THREADS), 0, (hipStream_t)stream, a);
      const hipError_t e = hipGetLastError();
      if (e != hipSuccess) return (int)e;
    }
  }
  StepArgs a = {};
  const double c1 = 1.0 - __builtin_pow(beta1, (double)step), c2 = 1.0 - __builtin_pow(beta2, (double)step);
  a.b1 = beta1;
  a.b1_rest = 1.0 - beta1;
  a.b2 = beta2;
  a.b2_rest = 1.0 - beta2;
  a.keep = (float)(1.0 - rate * weight_decay);
  a.rate = (float)(rate / c1);
  a.root = (float)(1.0 / __builtin_sqrt(c2));
  a.eps = (float)eps;
  a.max_norm = max_norm;
  if (max_norm > 0.0 && parts) {
    a.partial = workspace;
    a.partials = (int)parts;
    a.norm = norm;
  }
  const uint32_t key = host_mixed(host_mixed((uint32_t)seed) + (uint32_t)step);
  for (int64_t first = 0; first < count;) {
    first += take(a, tensors, first, count, bits, key, false);
    if (!a.n) continue;
    const dim3 grid(std::min<uint32_t>(a.chunks, 2048));
    if (bits == 8) hipLaunchKernelGGL(adamw_step<true>, grid, dim3(THREADS), 0, (hipStream_t)stream, a);
    else hipLaunchKernelGGL(adamw_step<false>, grid, dim3(THREADS), 0, (hipStream_t)stream, a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return (int)e;
  }
  return QA_OK;
}

int qutai_amd_adamw_moments(const void* first, const void* second, const void* exponents, float* first_out,
                            float* second_out, int64_t count, void* stream) {
  if (count < 0 || count > (1ll << 42)) return QA_EINVAL;
  if (!count) return QA_OK;
  if (!first || !second || !exponents || !first_out || !second_out) return QA_EINVAL;
  const unsigned grid = (unsigned)std::min<int64_t>((count + THREADS - 1) / THREADS, 1 << 16);
  hipLaunchKernelGGL(adamw_moments, dim3(grid), dim3(THREADS), 0, (hipStream_t)stream, (const uint8_t*)first,
                     (const uint8_t*)second, (const int8_t*)exponents, first_out, second_out, count);
  return (int)hipGetLastError();
}

}  // extern "C"
