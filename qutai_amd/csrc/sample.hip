// One token per row of logits: C ABI `qutai_amd_sample`.
//
// With l_max a row's largest logit and T its temperature, token i weighs
//   w_i = exp((l_i - l_max) / T)   (64 bits).
// Tokens in the order of falling logits (equal ones: lowest index first):
//   top_k keeps the first k; top_p of those the shortest prefix that holds p of
//   their weight; min_p of those the ones with w_i >= min_p.
// The given number u picks the first token, in the order of indices, at which the
// running sum of the kept weights exceeds u times their sum.
//
// What is kept is a threshold on a logit's key (its bits, in an order of unsigned
// integers) and, among the tokens that lie on it, a number of them from the
// lowest index on: nothing is sorted.  The threshold is found digit by digit, from
// histograms of counts (top_k) or of weights (top_p).  Weights in a histogram are
// 64-bit integers, w_i 2^(62 - log2 vocab): their sums are exact, in any order.
#include "common.h"
#include "qutai_amd.h"

#include <initializer_list>

using namespace qa;

namespace {

constexpr int THREADS = 1024, WAVES = THREADS / 64;
constexpr int64_t VOCAB_LIMIT = 1 << 20;
constexpr int BINS = 2048;

struct SampleArgs {
  const void* logits;
  const void* uniforms;
  int64_t* tokens;
  float* probabilities;
  const float* temperatures;
  const int64_t* top_ks;
  const float* top_ps;
  const float* min_ps;
  double temperature, top_p, min_p;
  int64_t top_k;
  int vocab, wide_uniforms, vector, fraction;  // fraction: bits of a weight in a histogram
};

// Keys: larger for larger logits, equal for equal ones (both zeros, every NaN
// with -inf); 0 is below all of them.
template <class T> struct Key;
template <> struct Key<float> {
  static constexpr int E = 4, BITS = 32;
  static __device__ __forceinline__ uint32_t of(uint32_t bits) {
    float v = __uint_as_float(bits);
    v = v == v ? v + 0.f : -INFINITY;
    const uint32_t u = __float_as_uint(v);
    return u ^ ((int32_t)u < 0 ? 0xffffffffu : 0x80000000u);
  }
  static __device__ __forceinline__ float value(uint32_t key) {
    return __uint_as_float(key ^ ((int32_t)key < 0 ? 0x80000000u : 0xffffffffu));
  }
};
template <> struct Key<bf16_t> {
  static constexpr int E = 8, BITS = 16;
  static __device__ __forceinline__ uint32_t of(uint32_t bits) { return Key<float>::of(bits << 16) >> 16; }
  static __device__ __forceinline__ float value(uint32_t key) {
    return __uint_as_float(((key ^ (key & 0x8000u ? 0x8000u : 0xffffu)) & 0xffffu) << 16);
  }
};

template <class T>
struct Row {
  static constexpr int E = Key<T>::E;
  const T* p;
  int vocab, vector;
  __device__ __forceinline__ int steps() const { return (vocab + THREADS * E - 1) / (THREADS * E); }
  // the keys of tokens (step THREADS + thread) E .. + E; 0 behind the last
  __device__ __forceinline__ void keys(int step, uint32_t (&k)[E]) const {
    const int first = (step * THREADS + (int)threadIdx.x) * E;
    if (vector && first + E <= vocab) {
      const u32x4 w = global_load<u32x4>(p + first);
#pragma unroll
      for (int e = 0; e < E; e++) {
        if constexpr (E == 4) k[e] = Key<T>::of(w[e]);
        else k[e] = Key<T>::of((w[e >> 1] >> (16 * (e & 1))) & 0xffffu);
      }
    } else {
#pragma unroll
      for (int e = 0; e < E; e++) {
        k[e] = 0;
        if (first + e < vocab) {
          if constexpr (E == 4) k[e] = Key<T>::of(__float_as_uint(p[first + e]));
          else k[e] = Key<T>::of(p[first + e]);
        }
      }
    }
  }
};

struct Shared {
  union {
    uint32_t counts[BINS];
    unsigned long long masses[BINS];
    double sums[VOCAB_LIMIT / (THREADS * 4) * WAVES];  // kept weights of each step and wave
  };
  uint32_t ties[VOCAB_LIMIT / (THREADS * 4) * WAVES];
  unsigned long long part[WAVES];
  double wide[WAVES];
  unsigned long long found[3];
  int chosen;
};

template <class T>
__device__ __forceinline__ double weight(uint32_t key, float top, double scale) {
  const float l = Key<T>::value(key);
  if (l == top) return 1.0;
  const double behind = (double)top - (double)l;
  return behind < INFINITY ? exp(-behind * scale) : 0.0;
}

// The bin, from the top, at which a running sum of bins reaches `target` (> 0, at
// most their sum); found: bin, sum of the bins above it, its own value.  Threads
// take neighbouring bins, the highest first.
template <class V>
__device__ __forceinline__ void find_bin(Shared& s, const V* bins, unsigned long long target) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, high = BINS - 1 - 2 * (int)threadIdx.x;
  const unsigned long long a = bins[high], b = bins[high - 1];
  unsigned long long run = a + b;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const unsigned long long other = __shfl_up(run, o);
    if (lane >= o) run += other;
  }
  if (lane == 63) s.part[wave] = run;
  __syncthreads();
  for (int w = 0; w < wave; w++) run += s.part[w];
  const unsigned long long above = run - a - b;
  if (above < target && above + a >= target) s.found[0] = high, s.found[1] = above, s.found[2] = a;
  else if (above + a < target && run >= target) s.found[0] = high - 1, s.found[1] = above + a, s.found[2] = b;
  __syncthreads();
}

template <class T>
__global__ void __launch_bounds__(THREADS) sample_rows(SampleArgs a) {
  constexpr int E = Key<T>::E, KEY = Key<T>::BITS;
  __shared__ Shared s;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t r = blockIdx.x;
  const Row<T> row = {(const T*)a.logits + r * a.vocab, a.vocab, a.vector};
  const int steps = row.steps();
  const double temperature = a.temperatures ? (double)a.temperatures[r] : a.temperature;
  const int64_t top_k = a.top_ks ? a.top_ks[r] : a.top_k;
  const double top_p = a.top_ps ? (double)a.top_ps[r] : a.top_p;
  const double asked = a.min_ps ? (double)a.min_ps[r] : a.min_p, min_p = asked <= 1.0 ? asked : 1.0;

  // ---- the largest key and its lowest index
  uint32_t k[E], best = 0;
  int at = 0;
  for (int step = 0; step < steps; step++) {
    row.keys(step, k);
#pragma unroll
    for (int e = 0; e < E; e++)
      if (k[e] > best) best = k[e], at = (step * THREADS + tid) * E + e;
  }
  unsigned long long both = (unsigned long long)best << 32 | (0xffffffffu - (uint32_t)at);
#pragma unroll
  for (int o = 32; o; o >>= 1) {
    const unsigned long long other = __shfl_xor(both, o);
    both = other > both ? other : both;
  }
  if (lane == 0) s.part[wave] = both;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < WAVES; w++) both = s.part[w] > both ? s.part[w] : both;
  __syncthreads();
  const uint32_t top_key = (uint32_t)(both >> 32);
  const int top_at = (int)(0xffffffffu - (uint32_t)both);
  const float top = Key<T>::value(top_key);
  const bool none = top == -INFINITY;
  if (none || !(temperature > 0.0)) {
    if (tid == 0) {
      a.tokens[r] = none ? -1 : top_at;
      a.probabilities[r] = none ? 0.f : 1.f;
    }
    return;
  }
  const double scale = 1.0 / temperature;

  // ---- the threshold: keys above it are kept, and `keep` of the `tied` on it
  uint32_t threshold = 0;
  unsigned long long keep = 0, tied = 0;
  const bool by_count = top_k > 0 && top_k < a.vocab, by_mass = top_p < 1.0;
  constexpr int FIRST = KEY == 32 ? 21 : 5;  // digits of 11, 11 and 10 bits, or 11 and 5
  if (by_count) {
    unsigned long long wanted = (unsigned long long)top_k;
    uint32_t prefix = 0;
    for (int low = FIRST, width = 11, done = 0;;) {
      for (int i = tid; i < BINS; i += THREADS) s.counts[i] = 0;
      __syncthreads();
      for (int step = 0; step < steps; step++) {
        row.keys(step, k);
#pragma unroll
        for (int e = 0; e < E; e++)
          if (done == 0 || k[e] >> (KEY - done) == prefix) atomicAdd(&s.counts[(k[e] >> low) & ((1u << width) - 1)], 1u);
      }
      __syncthreads();
      find_bin(s, s.counts, wanted);
      prefix = prefix << width | (uint32_t)s.found[0];
      wanted -= s.found[1];
      tied = s.found[2];
      done += width;
      __syncthreads();
      if (low == 0) break;
      width = low < 11 ? low : low - 10 < 11 ? low - 10 : 11;
      low -= width;
    }
    threshold = prefix, keep = wanted;
  }
  const double unit = (double)(1ull << a.fraction);
  if (by_mass) {
    unsigned long long target = 0, above = 0, mass = 0;
    uint32_t prefix = 0;
    for (int low = FIRST, width = 11, done = 0;;) {
      for (int i = tid; i < BINS; i += THREADS) s.masses[i] = 0;
      __syncthreads();
      for (int step = 0; step < steps; step++) {
        row.keys(step, k);
#pragma unroll
        for (int e = 0; e < E; e++) {
          if (k[e] == 0 || k[e] < threshold || (by_count && k[e] == threshold)) continue;
          if (done == 0 || k[e] >> (KEY - done) == prefix)
            atomicAdd(&s.masses[(k[e] >> low) & ((1u << width) - 1)],
                      (unsigned long long)(weight<T>(k[e], top, scale) * unit + 0.5));
        }
      }
      if (by_count && tid == 0 && (done == 0 || threshold >> (KEY - done) == prefix))
        atomicAdd(&s.masses[(threshold >> low) & ((1u << width) - 1)],
                  keep * (unsigned long long)(weight<T>(threshold, top, scale) * unit + 0.5));
      __syncthreads();
      if (done == 0) {
        unsigned long long total = s.masses[2 * tid] + s.masses[2 * tid + 1];
#pragma unroll
        for (int o = 32; o; o >>= 1) total += __shfl_xor(total, o);
        if (lane == 0) s.part[wave] = total;
        __syncthreads();
        total = 0;
        for (int w = 0; w < WAVES; w++) total += s.part[w];
        __syncthreads();
        const double wanted = ceil(top_p * (double)total);
        target = wanted < 1.0 ? 1ull : (unsigned long long)wanted;
        target = target > total ? total : target;
      }
      find_bin(s, s.masses, target - above);
      prefix = prefix << width | (uint32_t)s.found[0];
      above += s.found[1];
      mass = s.found[2];
      done += width;
      __syncthreads();
      if (low == 0) break;
      width = low < 11 ? low : low - 10 < 11 ? low - 10 : 11;
      low -= width;
    }
    // the tokens on the threshold weigh the same
    const unsigned long long each = (unsigned long long)(weight<T>(prefix, top, scale) * unit + 0.5);
    tied = by_count && prefix == threshold ? tied : mass / each;
    keep = (target - above + each - 1) / each;
    threshold = prefix;
  }

  // ---- where tokens on the threshold are left out: how many lie before each step's wave
  const bool cut = (by_count || by_mass) && keep < tied;
  const int slots = steps * WAVES;
  if (cut) {
    for (int step = 0; step < steps; step++) {
      row.keys(step, k);
      int n = 0;
#pragma unroll
      for (int e = 0; e < E; e++) n += __popcll(__ballot(k[e] == threshold));
      if (lane == 0) s.ties[step * WAVES + wave] = n;
    }
    __syncthreads();
    if (wave == 0) {
      uint32_t before = 0;
      for (int i0 = 0; i0 < slots; i0 += 64) {
        const uint32_t n = i0 + lane < slots ? s.ties[i0 + lane] : 0;
        uint32_t run = n;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
          const uint32_t other = __shfl_up(run, o);
          if (lane >= o) run += other;
        }
        if (i0 + lane < slots) s.ties[i0 + lane] = before + run - n;
        before += __shfl(run, 63);
      }
    }
    __syncthreads();
  }

  // the kept weights of this thread's tokens of a step
  auto kept = [&](int step, double (&w)[E]) {
    row.keys(step, k);
    unsigned long long rank = 0;
    if (cut) {
      rank = s.ties[step * WAVES + wave];
#pragma unroll
      for (int e = 0; e < E; e++) {
        const unsigned long long on = __ballot(k[e] == threshold);
        rank += __popcll(on & ((1ull << lane) - 1));
      }
    }
#pragma unroll
    for (int e = 0; e < E; e++) {
      bool in = k[e] != 0 && k[e] >= threshold;
      if (cut && k[e] == threshold) in = rank++ < keep;
      w[e] = 0.0;
      if (in) {
        w[e] = weight<T>(k[e], top, scale);
        if (w[e] < min_p) w[e] = 0.0;
      }
    }
  };

  // ---- their sums, step by step and wave by wave (the order of indices)
  for (int step = 0; step < steps; step++) {
    double w[E], sum = 0.0;
    kept(step, w);
#pragma unroll
    for (int e = 0; e < E; e++) sum += w[e];
#pragma unroll
    for (int o = 32; o; o >>= 1) sum += __shfl_xor(sum, o);
    if (lane == 0) s.sums[step * WAVES + wave] = sum;
  }
  __syncthreads();
  if (wave == 0) {
    double before = 0.0;
    unsigned long long adds = 0;  // bit i0 / 64: this lane's sum there is not zero
    for (int i0 = 0; i0 < slots; i0 += 64) {
      double run = i0 + lane < slots ? s.sums[i0 + lane] : 0.0;
      if (run > 0.0) adds |= 1ull << (i0 / 64);
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) {
        const double other = __shfl_up(run, o);
        if (lane >= o) run += other;
      }
      run += before;
      if (i0 + lane < slots) s.sums[i0 + lane] = run;
      before = __shfl(run, 63);
    }
    // the first step and wave whose running sum exceeds u times the whole sum; else the last with a kept token
    const double all = before;
    double u = a.wide_uniforms ? ((const double*)a.uniforms)[r] : (double)((const float*)a.uniforms)[r];
    u = u > 0.0 ? (u < 1.0 ? u : 1.0) : 0.0;
    const double goal = u * all;
    int first = slots, last = 0;
    for (int i = lane; i < slots; i += 64) {
      if (!(adds >> (i / 64) & 1)) continue;
      if (first == slots && s.sums[i] > goal) first = i;
      last = i;
    }
#pragma unroll
    for (int o = 32; o; o >>= 1) {
      const int f = __shfl_xor(first, o), l = __shfl_xor(last, o);
      first = f < first ? f : first;
      last = l > last ? l : last;
    }
    if (lane == 0) {
      s.chosen = first < slots ? first : last;
      s.wide[0] = goal, s.wide[1] = all;
    }
  }
  __syncthreads();
  const int chosen = s.chosen;
  if (wave != chosen % WAVES) return;
  const double goal = s.wide[0], all = s.wide[1];
  double w[E], sum = 0.0;
  kept(chosen / WAVES, w);
#pragma unroll
  for (int e = 0; e < E; e++) sum += w[e];
  double run = sum;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const double other = __shfl_up(run, o);
    if (lane >= o) run += other;
  }
  const double base = chosen ? s.sums[chosen - 1] : 0.0;
  const unsigned long long over = __ballot(sum > 0.0 && base + run > goal), any = __ballot(sum > 0.0);
  const int owner = over ? __ffsll(over) - 1 : 63 - __clzll(any);
  if (lane != owner) return;
  double walk = base + run - sum, weigh = 0.0;
  int token = -1;
#pragma unroll
  for (int e = 0; e < E; e++) {
    if (w[e] > 0.0 && !(token >= 0 && walk > goal)) token = (chosen / WAVES * THREADS + tid) * E + e, weigh = w[e];
    walk += w[e];
  }
  a.tokens[r] = token;
  a.probabilities[r] = (float)(weigh / all);
}

}  // namespace

extern "C" int qutai_amd_sample(const void* logits, const void* uniforms, int64_t* tokens, float* probabilities,
                                int64_t rows, int64_t vocab, const float* temperatures, double temperature,
                                const int64_t* top_ks, int64_t top_k, const float* top_ps, double top_p,
                                const float* min_ps, double min_p, int dtype, int uniform_dtype, void* stream_) {
  if (rows < 0 || rows > (1 << 22) - 1 || vocab <= 0 || vocab > VOCAB_LIMIT) return QA_EINVAL;
  if ((dtype != BF16 && dtype != F32) || (uniform_dtype != F32 && uniform_dtype != F64)) return QA_EINVAL;
  if (!(temperature >= 0.0) || temperature > 1.7e308 || top_k < 0 || !(top_p >= 0.0) || !(min_p >= 0.0) || min_p > 1.0) return QA_EINVAL;
  if (rows == 0) return QA_OK;
  for (const void* p : {logits, uniforms, (const void*)tokens, (const void*)probabilities})
    if (!p) return QA_EINVAL;
  int log2 = 0;
  while ((1ll << log2) < vocab) log2++;
  const int es = dtype == BF16 ? 2 : 4;
  const SampleArgs a = {logits, uniforms, tokens, probabilities, temperatures, top_ks, top_ps, min_ps, temperature,
                        top_p, min_p, top_k, (int)vocab, uniform_dtype == F64, (uintptr_t)logits % 16 == 0 && vocab * es % 16 == 0,
                        62 - log2};
  hipStream_t stream = (hipStream_t)stream_;
  if (dtype == BF16) hipLaunchKernelGGL(sample_rows<bf16_t>, dim3((unsigned)rows), dim3(THREADS), 0, stream, a);
  else hipLaunchKernelGGL(sample_rows<float>, dim3((unsigned)rows), dim3(THREADS), 0, stream, a);
  return (int)hipGetLastError();
}
