// One AdamW step over many tensors: C ABI `qutai_amd_adamw`, `_workspace`, `_moments`.
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
// are computed in 64 bits, so that codes are those of the definition whatever the order
// of operations, and fp32's are rounded once.
//
// A block with an infinity, a NaN or a moment of 2^127 or more has the exponent 127 and
// reads as NaN, so the next step makes NaN of all 256 parameters (the codes have none for a
// single value; without a norm to find it by, a gradient that is not finite is the caller's).
//
// One launch steps 48 tensors, whose records are its arguments: a workgroup takes 1024 or
// 4096 values of one of them at a time, with 8 bits a wave a block.  Memory bounds it
// where parameters are fp32 (61 million values in 20 tensors: 32-bit moments 290 us for 1.7
// GB, 5.9 TB/s; 8 bits 205 for 973 MB, 4.7 TB/s, and 36 for the norm of 243 MB); 5 million
// bf16 values in 17 tensors with moments of 8 bits take 17.5 us for 50 MB, bound by about
// 90 vector instructions a value, an eighth of them in 64 bits.
#include "common.h"
#include "qutai_amd.h"

#include <algorithm>
#include <cfloat>

using namespace qa;

namespace {

constexpr int THREADS = 256, BLOCK = 256;     // BLOCK: values that share an exponent
constexpr int NORM_CHUNK = 4096;              // values of a workgroup's turn of the norm
constexpr int NORM_GROUPS = 1024;             // partial sums of a launch
constexpr int TENSORS = 48;                   // of a launch: their records fit the kernel's arguments
constexpr int NOT_FINITE = 127;

// Values of a workgroup's turn of the step, and workgroups of a launch at most.  Moments
// of 8 bits: a block for each wave.  fp32 moments: four loads of every array in flight
// where there are turns enough for the GPU, shorter turns of more workgroups else.  us with
// turns of 1024, 2048 and 4096: 61 million values, 8 bits 203, 205 and 225, fp32 351, 323
// and 310; 15 million, fp32, 78 and 75 (1024, 4096), 4 million 17.9 and 18.9, 1 million 5.3
// and 8.8; 5 million bf16 values, 8 bits, 17.6, 18.0 and 20.6.  With 16384 workgroups
// instead of 2048 the 61 million take 290 instead of 309 (fp32) and 217 instead of 207.
// (The norm: 53, 38 and 36.)
constexpr int SHORT_CHUNK = 1024, LONG_CHUNK = 4096, SHORT_GROUPS = 2048, LONG_GROUPS = 16384;
constexpr int64_t LONG_FROM = 1ll << 23;  // values of all tensors

struct Tensor {
  void* p;
  const void* g;
  void* m;
  void* v;
  int8_t* e;
  int64_t count;
  uint32_t chunks;  // of the tensors before it in this launch
  uint32_t key;     // of its rounding
  int bf16, whole;  // whole: every address is a multiple of 16 bytes
};

struct StepArgs {
  int n;
  uint32_t chunks;
  double b1, b1_rest, b2, b2_rest;
  float decay, rate, root, eps;  // lr times the decay, lr / c1, 1 / sqrt(c2)
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

// The record that holds chunk c: the last whose first chunk is not behind it.
// `starts`: lane i's is record i's first chunk.
template <class Args>
__device__ __forceinline__ uint32_t starts_of(const Args& a) {
  const int lane = threadIdx.x & 63;
  return lane < a.n ? a.t[lane].chunks : 0xffffffffu;
}
__device__ __forceinline__ int tensor_of(uint32_t starts, uint32_t c) {
  return __builtin_popcountll(__builtin_amdgcn_ballot_w64(starts <= c)) - 1;
}

// Four values from index i on, and back: at once where `whole` (i a multiple of 4),
// else one by one, those at or beyond `end` left out.
template <class T>
__device__ __forceinline__ f32x4 get4(const void* x, int64_t i, int64_t end, bool whole) {
  const T* p = (const T*)x + i;
  f32x4 v = {};
  if (whole) {
    if constexpr (sizeof(T) == 4) {
      v = global_load_nt<f32x4>(p);
    } else {
      const u32x2 w = global_load_nt<u32x2>(p);
      v = f32x4{__uint_as_float(w[0] << 16), __uint_as_float(w[0] & 0xffff0000u), __uint_as_float(w[1] << 16),
                __uint_as_float(w[1] & 0xffff0000u)};
    }
  } else {
#pragma unroll
    for (int j = 0; j < 4; j++)
      if (i + j < end) {
        if constexpr (sizeof(T) == 4) v[j] = p[j];
        else v[j] = bf16_to_f32(p[j]);
      }
  }
  return v;
}
template <class T>
__device__ __forceinline__ void put4(void* x, int64_t i, int64_t end, bool whole, const f32x4& v) {
  T* p = (T*)x + i;
  if (whole) {
    if constexpr (sizeof(T) == 4) global_store_nt(p, v);
    else global_store_nt(p, u32x2{pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3])});
  } else {
#pragma unroll
    for (int j = 0; j < 4; j++)
      if (i + j < end) {
        if constexpr (sizeof(T) == 4) p[j] = v[j];
        else p[j] = f32_to_bf16(v[j]);
      }
  }
}
__device__ __forceinline__ uint32_t get_codes(const void* x, int64_t i, int64_t end, bool whole) {
  const uint8_t* p = (const uint8_t*)x + i;
  if (whole) return global_load_nt<uint32_t>(p);
  uint32_t w = 0;
#pragma unroll
  for (int j = 0; j < 4; j++)
    if (i + j < end) w |= (uint32_t)p[j] << 8 * j;
  return w;
}
__device__ __forceinline__ void put_codes(void* x, int64_t i, int64_t end, bool whole, uint32_t w) {
  uint8_t* p = (uint8_t*)x + i;
  if (whole) {
    global_store_nt(p, w);
  } else {
#pragma unroll
    for (int j = 0; j < 4; j++)
      if (i + j < end) p[j] = (uint8_t)(w >> 8 * j);
  }
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

template <class T>
__device__ __forceinline__ void square_sum(const Tensor& t, int64_t start, int64_t end, double& sum) {
  constexpr int TURNS = NORM_CHUNK / (4 * THREADS);  // a thread takes 4 values, and 4 more a thousand on
  f32x4 g[TURNS];
  const int64_t i = start + 4 * threadIdx.x;
#pragma unroll
  for (int u = 0; u < TURNS; u++) {
    const int64_t at = i + 4 * THREADS * u;
    g[u] = get4<T>(t.g, at, end, t.whole && at + 4 <= end);
  }
#pragma unroll
  for (int u = 0; u < TURNS; u++)
#pragma unroll
    for (int j = 0; j < 4; j++) sum = fma((double)g[u][j], (double)g[u][j], sum);
}

__global__ void __launch_bounds__(THREADS) adamw_norm(NormArgs a) {
  __shared__ double shared[4];
  double sum = 0.0;
  const uint32_t starts = starts_of(a);
  for (uint32_t c = blockIdx.x; c < a.chunks; c += gridDim.x) {
    const Tensor& t = a.t[tensor_of(starts, c)];
    const int64_t start = (int64_t)(c - t.chunks) * NORM_CHUNK, end = min(t.count, start + NORM_CHUNK);
    if (t.bf16) square_sum<bf16_t>(t, start, end, sum);
    else square_sum<float>(t, start, end, sum);
  }
  sum = group_sum(sum, shared);
  if (threadIdx.x == 0) a.partial[blockIdx.x] = sum;
}

__host__ __device__ __forceinline__ uint32_t mixed(uint32_t x) {
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

// The code of a magnitude: in steps of an eighth of its binade (of the lowest one
// where it lies below), with 16 bits of a step's rest; those bits decide with `bits`
// whether it is rounded up.
__device__ __forceinline__ uint32_t coded(double magnitude, int least, uint32_t bits) {
  const int mine = max((int)(high_word(magnitude) >> 20 & 0x7ff) - 1023, least);
  return (uint32_t)(mine - least) * 8 + (((uint32_t)ldexp(magnitude, 19 - mine) + bits) >> 16);
}

// What a code's float of the same fields is multiplied by to be its value: a code's
// exponent and fraction, put into the lowest exponent bits and highest fraction bits of
// a float, are the code's value times 2^-126 / 2^L, the lowest binade's (whose codes
// are subnormal floats) included.
__device__ __forceinline__ double code_scale(int exponent, int below) {
  if (exponent == NOT_FINITE) return NAN;
  return __longlong_as_double((int64_t)(exponent - below + 126 + 1023) << 52);
}

// Maximum over a wave, the same in every lane: within rows of 16 lanes by
// data-parallel moves, across them by exchanges of rows and halves.
__device__ __forceinline__ uint32_t wave_max(uint32_t x) {
  x = max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0xB1, 0xf, 0xf, true));   // lanes 1 0 3 2
  x = max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x4E, 0xf, 0xf, true));   // lanes 2 3 0 1
  x = max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x141, 0xf, 0xf, true));  // half a row, reversed
  x = max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x140, 0xf, 0xf, true));  // a row, reversed
  const auto rows = __builtin_amdgcn_permlane16_swap(x, x, false, false);
  x = max((uint32_t)rows[0], (uint32_t)rows[1]);
  const auto halves = __builtin_amdgcn_permlane32_swap(x, x, false, false);
  return max((uint32_t)halves[0], (uint32_t)halves[1]);
}

// The 256 values from `base` on by a wave, four to a lane.
template <class T>
struct Block8 {
  f32x4 p, g;
  uint32_t m, v;
  int e1, e2;
  __device__ __forceinline__ void load(const Tensor& t, int64_t base, int64_t end, int lane) {
    const int64_t i = base + 4 * lane;
    const bool whole = t.whole && i + 4 <= end;
    g = get4<T>(t.g, i, end, whole);
    p = get4<T>(t.p, i, end, whole);
    m = get_codes(t.m, i, end, whole);
    v = get_codes(t.v, i, end, whole);
    if (base < end) {  // the wave's own block alone writes them
      e1 = t.e[base / BLOCK * 2];
      e2 = t.e[base / BLOCK * 2 + 1];
    }
  }
  __device__ __forceinline__ void step(const StepArgs& a, const Tensor& t, int64_t base, int64_t end, int lane, double factor) {
    if (base >= end) return;
    const int64_t i = base + 4 * lane;
    const bool whole = t.whole && i + 4 <= end;
    double m1[4], v1[4];
    uint32_t most1 = 0, most2 = 0;
    // a product with a power of two is exact, so the decay may take it
    const double d1 = a.b1 * code_scale(uniform32(e1), 14), d2 = a.b2 * code_scale(uniform32(e2), 30);
#pragma unroll
    for (int j = 0; j < 4; j++) {
#pragma clang fp contract(off)
      const uint32_t c1 = m >> 8 * j, c2 = v >> 8 * j;
      const float m0 = __uint_as_float((c1 & 127) << 20 | (c1 & 128) << 24), v0 = __uint_as_float((c2 & 255) << 20);
      const double gj = (double)g[j] * factor;
      m1[j] = d1 * (double)m0 + a.b1_rest * gj;
      v1[j] = d2 * (double)v0 + a.b2_rest * (gj * gj);
      // values behind the end are zeros, unless the block's exponent says NaN
      most1 = max(most1, high_word(m1[j]) & 0x7fffffffu);
      most2 = max(most2, high_word(v1[j]) & 0x7fffffffu);
    }
    const int E1 = uniform32(block_exponent(wave_max(most1))), E2 = uniform32(block_exponent(wave_max(most2)));
    uint32_t codes1 = 0, codes2 = 0;
    f32x4 p1;
    const uint32_t seed = (uint32_t)i * 0x9E3779B9u + t.key;
#pragma unroll
    for (int j = 0; j < 4; j++) {
      const uint32_t bits = mixed(seed + j * 0x9E3779B9u);
      codes1 |= (coded(fabs(m1[j]), E1 - 14, bits & 0xffff) | (high_word(m1[j]) >> 24 & 128)) << 8 * j;
      codes2 |= max(coded(v1[j], E2 - 30, bits >> 16), v1[j] > 0.0 ? 1u : 0u) << 8 * j;
      // the hardware's fp64 root holds fp32's bits for every value that fp64 holds
      const float root = (float)__builtin_amdgcn_sqrt(v1[j]);
      p1[j] = p[j] + fmaf(-a.decay, p[j], -a.rate * (float)m1[j] * __builtin_amdgcn_rcpf(fmaf(root, a.root, a.eps)));
    }
    if (E1 == NOT_FINITE) codes1 = 0;
    if (E2 == NOT_FINITE) codes2 = 0;
    put_codes(t.m, i, end, whole, codes1);
    put_codes(t.v, i, end, whole, codes2);
    put4<T>(t.p, i, end, whole, p1);
    if (lane == 0) {
      t.e[base / BLOCK * 2] = (int8_t)E1;
      t.e[base / BLOCK * 2 + 1] = (int8_t)E2;
    }
  }
};

template <class T, int CHUNK>
__device__ __forceinline__ void step8(const StepArgs& a, const Tensor& t, int64_t start, int64_t end, double factor) {
  const int lane = threadIdx.x & 63, wave = uniform32(threadIdx.x >> 6);
  constexpr int N = CHUNK / BLOCK / (THREADS / 64);  // blocks of a wave, whose loads go out together
  Block8<T> b[N];
#pragma unroll
  for (int u = 0; u < N; u++) b[u].load(t, start + (u * (THREADS / 64) + wave) * BLOCK, end, lane);
#pragma unroll
  for (int u = 0; u < N; u++) b[u].step(a, t, start + (u * (THREADS / 64) + wave) * BLOCK, end, lane, factor);
}

template <class T, int CHUNK>
__device__ __forceinline__ void step32(const StepArgs& a, const Tensor& t, int64_t start, int64_t end, double factor) {
#pragma clang fp contract(off)
  constexpr int TURNS = CHUNK / (4 * THREADS);
  f32x4 g[TURNS], p[TURNS], m[TURNS], v[TURNS];
#pragma unroll
  for (int u = 0; u < TURNS; u++) {
    const int64_t i = start + 4 * (threadIdx.x + THREADS * u);
    const bool whole = t.whole && i + 4 <= end;
    g[u] = get4<T>(t.g, i, end, whole);
    p[u] = get4<T>(t.p, i, end, whole);
    m[u] = get4<float>(t.m, i, end, whole);
    v[u] = get4<float>(t.v, i, end, whole);
  }
#pragma unroll
  for (int u = 0; u < TURNS; u++) {
    const int64_t i = start + 4 * (threadIdx.x + THREADS * u);
    const bool whole = t.whole && i + 4 <= end;
#pragma unroll
    for (int j = 0; j < 4; j++) {
      // memory bounds the step: moments in 64 bits, rounded once
      const double gj = (double)g[u][j] * factor;
      m[u][j] = (float)fma(a.b1, (double)m[u][j], a.b1_rest * gj);
      v[u][j] = (float)fma(a.b2, (double)v[u][j], a.b2_rest * (gj * gj));
      p[u][j] += fmaf(-a.decay, p[u][j], -a.rate * (m[u][j] / fmaf(sqrtf(v[u][j]), a.root, a.eps)));
    }
    put4<float>(t.m, i, end, whole, m[u]);
    put4<float>(t.v, i, end, whole, v[u]);
    put4<T>(t.p, i, end, whole, p[u]);
  }
}

template <bool EIGHT, int CHUNK>
__global__ void __launch_bounds__(THREADS) adamw_step(StepArgs a) {
  __shared__ double shared[4];
  const uint32_t starts = starts_of(a);
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
    const Tensor& t = a.t[tensor_of(starts, c)];
    const int64_t start = (int64_t)(c - t.chunks) * CHUNK, end = min(t.count, start + CHUNK);
    if constexpr (EIGHT) {
      if (t.bf16) step8<bf16_t, CHUNK>(a, t, start, end, factor);
      else step8<float, CHUNK>(a, t, start, end, factor);
    } else {
      if (t.bf16) step32<bf16_t, CHUNK>(a, t, start, end, factor);
      else step32<float, CHUNK>(a, t, start, end, factor);
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

// Records of up to TENSORS tensors from `first` on, in turns of `chunk` values; returns
// how many tensors they took (those without values among them).
template <class Args>
int64_t take(Args& a, const int64_t* tensors, int64_t first, int64_t count, uint32_t key, int64_t chunk) {
  a.n = 0;
  a.chunks = 0;
  int64_t i = first;
  for (; i < count && a.n < TENSORS; i++) {
    const int64_t* r = tensors + 8 * i;
    if (r[5] == 0) continue;
    const int64_t chunks = (r[5] + chunk - 1) / chunk;  // below 2^31: valid()
    if (a.chunks + chunks > 0x7fffffff) break;
    Tensor& t = a.t[a.n++];
    t.p = (void*)r[0];
    t.g = (const void*)r[1];
    t.m = (void*)r[2];
    t.v = (void*)r[3];
    t.e = (int8_t*)r[4];
    t.count = r[5];
    t.chunks = a.chunks;
    t.bf16 = r[6] == BF16;
    t.whole = (r[0] | r[1] | r[2] | r[3]) % 16 == 0;
    t.key = mixed(key + (uint32_t)r[7]);
    a.chunks += (uint32_t)chunks;
  }
  return i - first;
}

// Launches that any `tensors` tensors of `values` values need at most: one ends with
// TENSORS of them, or with 2^30 chunks at least.
int64_t launches(int64_t tensors, int64_t values) {
  return (tensors + TENSORS - 1) / TENSORS + ((values / NORM_CHUNK + tensors) >> 30);
}

bool valid(const int64_t* tensors, int64_t count, int bits, int64_t& values) {
  values = 0;
  if (count < 0 || count > 1 << 24 || (count && !tensors)) return false;
  for (int64_t i = 0; i < count; i++) {
    const int64_t* r = tensors + 8 * i;
    if (r[5] < 0 || r[5] > (1ll << 40) || (r[6] != F32 && r[6] != BF16)) return false;
    if (r[5] == 0) continue;
    values += r[5];
    if (values > 1ll << 48) return false;
    if (!r[1] || r[1] % (r[6] == BF16 ? 2 : 4)) return false;
    if (!r[0] || r[0] % (r[6] == BF16 ? 2 : 4) || !r[2] || !r[3]) return false;
    if (bits == 8 ? !r[4] : r[2] % 4 || r[3] % 4) return false;
  }
  return true;
}

}  // namespace

extern "C" {

int64_t qutai_amd_adamw_workspace(int64_t count, int64_t values) {
  return count < 0 || count > 1 << 24 || values < 0 || values > 1ll << 48 ? 0 : launches(count, values) * NORM_GROUPS;
}

int qutai_amd_adamw(const int64_t* tensors, int64_t count, int bits, double rate, double beta1, double beta2,
                    double eps, double weight_decay, int64_t step, uint64_t seed, double max_norm, double* workspace,
                    int64_t workspace_values, double* norm, void* stream) {
  int64_t values;
  if ((bits != 8 && bits != 32) || !valid(tensors, count, bits, values)) return QA_EINVAL;
  if (!(beta1 >= 0.0 && beta1 < 1.0 && beta2 >= 0.0 && beta2 < 1.0) || step < 1) return QA_EINVAL;
  if (!(rate >= 0.0) || !(rate < 1e30) || !(weight_decay >= 0.0) || !(weight_decay < 1e30) || !(max_norm >= 0.0))
    return QA_EINVAL;
  // The kernels take these in fp32: an eps that is 0 there, or whose reciprocal is infinite,
  // makes 0 / 0 of a value without a gradient, an infinite rate or decay inf * 0.
  const double c1 = 1.0 - __builtin_pow(beta1, (double)step), c2 = 1.0 - __builtin_pow(beta2, (double)step);
  if (!(eps >= FLT_MIN) || !(eps <= FLT_MAX) || !(rate / c1 <= FLT_MAX) || !(rate * weight_decay <= FLT_MAX)) return QA_EINVAL;
  int64_t parts = 0;
  if (max_norm > 0.0 && values) {
    if (!workspace || (uintptr_t)workspace % 8 || workspace_values < launches(count, values) * NORM_GROUPS) return QA_EWORKSPACE;
    NormArgs a = {};
    for (int64_t first = 0; first < count;) {
      first += take(a, tensors, first, count, 0, NORM_CHUNK);
      if (!a.n) continue;
      a.partial = workspace + parts;
      const unsigned groups = std::min<uint32_t>(a.chunks, NORM_GROUPS);
      parts += groups;
      hipLaunchKernelGGL(adamw_norm, dim3(groups), dim3(THREADS), 0, (hipStream_t)stream, a);
      const hipError_t e = hipGetLastError();
      if (e != hipSuccess) return (int)e;
    }
  }
  StepArgs a = {};
  a.b1 = beta1;
  a.b1_rest = 1.0 - beta1;
  a.b2 = beta2;
  a.b2_rest = 1.0 - beta2;
  a.decay = (float)(rate * weight_decay);
  a.rate = (float)(rate / c1);
  a.root = (float)(1.0 / __builtin_sqrt(c2));
  a.eps = (float)eps;
  a.max_norm = max_norm;
  if (parts) {
    a.partial = workspace;
    a.partials = (int)parts;
    a.norm = norm;
  }
  const uint32_t key = mixed(mixed((uint32_t)seed) + (uint32_t)step);
  const bool longer = bits == 32 && values >= LONG_FROM;
  for (int64_t first = 0; first < count;) {
    first += take(a, tensors, first, count, key, longer ? LONG_CHUNK : SHORT_CHUNK);
    if (!a.n) continue;
    const dim3 grid(std::min<uint32_t>(a.chunks, longer ? LONG_GROUPS : SHORT_GROUPS));
    if (bits == 8) hipLaunchKernelGGL((adamw_step<true, SHORT_CHUNK>), grid, dim3(THREADS), 0, (hipStream_t)stream, a);
    else if (longer) hipLaunchKernelGGL((adamw_step<false, LONG_CHUNK>), grid, dim3(THREADS), 0, (hipStream_t)stream, a);
    else hipLaunchKernelGGL((adamw_step<false, SHORT_CHUNK>), grid, dim3(THREADS), 0, (hipStream_t)stream, a);
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
