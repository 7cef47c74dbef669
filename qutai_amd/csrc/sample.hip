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
// What is kept is a threshold on the logit and, among the tokens that lie on it, a
// number of them from the lowest index on: nothing is sorted.  A workgroup of 512
// threads owns a row and keeps its first 32 steps (of 16 bytes per thread: 131072
// bf16 or 65536 fp32 logits) in registers; what lies behind is read again by every
// pass.  A NaN, which no comparison lets through, stands behind the last token.
//  top_k: the k-th largest of the threads' maxima (two each) bounds the k-th largest logit
//  from below; the few logits from there on go into a list in LDS, where the
//  threshold is found.
//  top_p: weights in bins of 1/32 of a power of two, whose sums are 64-bit integers:
//  the same in any order.  They count each weight in units of 2^-45 of the largest
//  (2^-42 in 2^20 tokens), so the prefix may end one token off where a sum of more
//  bits lies within the roundings of its goal, and a top_p within some 2^-29 of 1 leaves
//  out tokens that weigh less than half a unit.
//  The logits of the bin that the prefix ends in go into the list.
// A list is searched digit by digit of its keys (bits in an order of unsigned
// integers), from histograms, a short one by comparing all with all.  Where it
// overflows (thousands of equal or nearly equal logits, or a large k) the whole row
// is searched.
// bf16 logits are counted by number instead: see Window.  Their weights are then a
// table, too.
//
// Bound by vector operations: one on each of a CU's 131072 logits takes 1.2 us, a
// weight some 20 of them.  200 rows of 131072 bf16 logits: 25 us for the largest
// alone, 45 without a filter, 48 with top_k 50, 64 with top_p .9 (passes over memory
// with a sorted digit search: 248); a row of 32768 fp32 logits with both: 27 us.
#include "common.h"
#include "qutai_amd.h"

#include <initializer_list>

using namespace qa;

namespace {

constexpr int THREADS = 512, WAVES = THREADS / 64;
constexpr int64_t VOCAB_LIMIT = 1 << 20;
constexpr int BINS = 2048, LIST = 4096, FEW = 192;
// bf16: exponents, and entries of a table with one for each number of these exponents (see Window)
constexpr int MAGNITUDES = 20 * 128, ENTRIES = 2 * MAGNITUDES + 4;
constexpr int SPAN = 8, HELD = 4 * SPAN;  // steps of a register vector, and of all of them

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
  int vocab, wide_uniforms, vector, fraction;  // fraction: bits of a weight in a bin
};

typedef uint32_t u32x32 __attribute__((ext_vector_type(4 * SPAN)));

// Larger for larger logits, equal for equal ones (both zeros); above 0 for all but NaN.
__device__ __forceinline__ uint32_t key_of(float v) {
  const uint32_t u = __float_as_uint(v + 0.f);
  return u ^ ((int32_t)u < 0 ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t key) {
  return __uint_as_float(key ^ ((int32_t)key < 0 ? 0x80000000u : 0xffffffffu));
}

struct Shared {
  union {
    struct {
      union {
        uint32_t counts[BINS];
        unsigned long long masses[BINS];
      };
      float list[LIST];
      uint32_t numbers[ENTRIES];
    };
    double sums[VOCAB_LIMIT / (THREADS * 4) * WAVES];  // kept weights of each step and wave
  };
  uint32_t ties[VOCAB_LIMIT / (THREADS * 4) * WAVES];
  double table[ENTRIES];  // bf16: the weight of each number
  double powers[32];  // 2^(-j / 32)
  unsigned long long part[WAVES];
  double wide[2];
  unsigned long long found[4];
  float bound[4];
  uint32_t listed;
  int chosen;
};

// Another lane's value by a data-parallel move (no trip through LDS): rows are of 16
// lanes; 0 where the source is none, or where row_mask leaves the row out.
template <int CTRL, int ROW_MASK = 0xf, class V>
__device__ __forceinline__ V moved(V x) {
  if constexpr (sizeof(V) == 4) {
    return __builtin_bit_cast(V, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), CTRL, ROW_MASK, 0xf, true));
  } else {
    u32x2 w = __builtin_bit_cast(u32x2, x);
#pragma unroll
    for (int i = 0; i < 2; i++) w[i] = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)w[i], CTRL, ROW_MASK, 0xf, true);
    return __builtin_bit_cast(V, w);
  }
}
// A running sum over a wave's lanes; the last lane has the whole (which is all that
// `wave_sum` is for: its other lanes mean nothing).
template <class V>
__device__ __forceinline__ V wave_scan(V x) {
  x += moved<0x111>(x);  // the lane 1, 2, 4 and 8 below, in its row
  x += moved<0x112>(x);
  x += moved<0x114>(x);
  x += moved<0x118>(x);
  x += moved<0x142, 0xa>(x);         // the last of the row below, for rows 1 and 3
  return x + moved<0x143, 0xc>(x);  // lane 31, for rows 2 and 3
}
template <class V>
__device__ __forceinline__ V wave_sum(V x) {
  x += moved<0xB1>(x);   // lane ^ 1
  x += moved<0x4E>(x);   // lane ^ 2
  x += moved<0x141>(x);  // mirrored in 8 lanes, then in 16
  x += moved<0x140>(x);
  x += moved<0x142, 0xa>(x);
  return x + moved<0x143, 0xc>(x);
}

// w = 2^(-t / 32), t = (top - l) 32 log2(e) / T: a table of 32 powers for the nearest
// integer n of t, and for the rest, at most half, a polynomial of degree four (the
// exponential's series up to the fifth power, that power economised: within 9e-14).
// Means nothing where t lies above 32000, or l is not finite: see `least_of`.
constexpr double ROUND = 6755399441055744.0;  // 1.5 2^52: adding it leaves an integer in the low bits

struct Weigh {
  const double* powers;
  double top, scale;
  __device__ __forceinline__ double behind(float l) const { return (top - (double)l) * scale; }
  __device__ __forceinline__ double operator()(float l, int& n) const {
    const double t = behind(l), whole = t + ROUND, x = t - (whole - ROUND);
    n = __double2loint(whole);
    double y = fma(x, 9.172562701824643e-09, -1.6938633902808837e-06);
    y = fma(x, y, 0.0002345961982022468);
    y = fma(x, y, -0.021660849391722175);
    y = fma(x, y, 1.0);
    y *= powers[n & 31];
    return __hiloint2double(__double2hiint(y) - ((n & ~31) << 15), __double2loint(y));  // times 2^-(n / 32)
  }
  __device__ __forceinline__ double operator()(float l) const {
    int n;
    return (*this)(l, n);
  }
};

// bf16 logits by number: entry MAGNITUDES + 3 + m for the m-th number of the window
// of exponents, from `lo` on, MAGNITUDES - m for its negative; between them two
// entries for what is smaller, zeros among it, at the ends two for what is larger.
typedef short s16x2 __attribute__((ext_vector_type(2)));
struct Window {
  int lo;  // bits of the smallest magnitude, 1 at least
  // the entries of a word's two logits; `small` gets a sign bit where one is below the window
  __device__ __forceinline__ s16x2 entries(uint32_t w, uint32_t& small) const {
    const s16x2 low = {(short)lo, (short)lo}, least = {-1, -1}, most = {MAGNITUDES, MAGNITUDES};
    const s16x2 bits = __builtin_bit_cast(s16x2, w), sign = bits >> 15;
    s16x2 m = __builtin_bit_cast(s16x2, w & 0x7fff7fffu) - low;
    m = __builtin_elementwise_min(__builtin_elementwise_max(m, least), most);
    small |= __builtin_bit_cast(uint32_t, m);
    const s16x2 middle = {MAGNITUDES + 3, MAGNITUDES + 3};
    return (m ^ sign) + sign + sign + middle;
  }
  __device__ __forceinline__ float value(int entry) const {
    const int m = entry >= MAGNITUDES + 3 ? entry - MAGNITUDES - 3 : MAGNITUDES - entry;
    return __uint_as_float((uint32_t)(lo + m) << 16 | (entry >= MAGNITUDES + 3 ? 0u : 0x80000000u));
  }
  __device__ __forceinline__ bool holds(int entry) const {
    return entry > 0 && entry < ENTRIES - 1 && entry != MAGNITUDES + 1 && entry != MAGNITUDES + 2;
  }
};

// The smallest logit (by a wave, all lanes) that `enough` accepts, which accepts
// every larger one up to top; 64 candidates at a time, of which the largest that
// is not enough is searched on.
template <class F>
__device__ __forceinline__ float least_of(float top, F enough) {
  const int lane = threadIdx.x & 63;
  uint32_t base = 0;
#pragma nounroll
  for (int shift = 26; shift >= 0; shift = shift == 2 ? 0 : shift - 6) {
    const uint32_t candidate = base + ((uint32_t)lane << shift);
    bool below = candidate == 0;
    if (candidate && candidate < key_of(top)) {
      const float l = value_of(candidate);
      below = !(l > -INFINITY) || !enough(l);
    }
    const unsigned long long lanes = __ballot(below && (shift || lane < 4));
    base += (uint32_t)(63 - __clzll(lanes)) << shift;
  }
  return value_of(base + 1);
}

// The bin, from the top, at which a running sum of bins reaches `target` (> 0, at
// most their sum); found: bin, sum of the bins above it, its own value.  Threads
// take neighbouring bins, the highest first.
template <class V>
__device__ __forceinline__ void find_bin(Shared& s, const V* bins, unsigned long long target) {
  constexpr int PER = BINS / THREADS;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, high = BINS - 1 - PER * (int)threadIdx.x;
  unsigned long long own[PER], run = 0;
#pragma unroll
  for (int i = 0; i < PER; i++) run += own[i] = bins[high - i];
  const unsigned long long mine = run;
  run = wave_scan(run);
  if (lane == 63) s.part[wave] = run;
  __syncthreads();
  unsigned long long before[WAVES];  // read together
#pragma unroll
  for (int w = 0; w < WAVES; w++) before[w] = s.part[w];
#pragma unroll
  for (int w = 0; w < WAVES; w++) run += w < wave ? before[w] : 0;
  if (run - mine < target && run >= target) {
    unsigned long long above = run - mine;
    int i = 0;
#pragma unroll
    for (int n = 0; n < PER - 1; n++)
      if (i == n && above + own[n] < target) above += own[n], i = n + 1;
    s.found[0] = high - i, s.found[1] = above;
    unsigned long long value = own[0];
#pragma unroll
    for (int n = 1; n < PER; n++) value = i == n ? own[n] : value;
    s.found[2] = value;
  }
  __syncthreads();
}

// The same over amount(entry) of the bf16 entries; target 0 is goal(their sum).
template <class F, class Goal>
__device__ __forceinline__ void find_entry(Shared& s, F amount, unsigned long long target, Goal goal) {
  constexpr int PER = (ENTRIES + THREADS - 1) / THREADS;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, high = ENTRIES - 1 - PER * (int)threadIdx.x;
  unsigned long long own[PER], run = 0;
#pragma unroll
  for (int i = 0; i < PER; i++) run += own[i] = high - i >= 0 ? amount(high - i) : 0;
  const unsigned long long mine = run;
  run = wave_scan(run);
  if (lane == 63) s.part[wave] = run;
  __syncthreads();
  unsigned long long before[WAVES], total = 0;
#pragma unroll
  for (int w = 0; w < WAVES; w++) before[w] = s.part[w];
#pragma unroll
  for (int w = 0; w < WAVES; w++) {
    run += w < wave ? before[w] : 0;
    total += before[w];
  }
  if (target == 0) target = goal(total);
  if (target > total) target = total;  // fewer numbers than top_k
  if (run - mine < target && run >= target) {
    unsigned long long above = run - mine;
    int i = 0;
#pragma unroll
    for (int n = 0; n < PER - 1; n++)
      if (i == n && above + own[n] < target) above += own[n], i = n + 1;
    s.found[0] = high - i, s.found[1] = above, s.found[3] = target;
  }
  __syncthreads();
}

template <class V>
__device__ __forceinline__ unsigned long long sum_bins(Shared& s, const V* bins) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  unsigned long long total = 0;
#pragma unroll
  for (int i = 0; i < BINS / THREADS; i++) total += bins[threadIdx.x + i * THREADS];
  total = wave_sum(total);
  if (lane == 63) s.part[wave] = total;
  __syncthreads();
  total = 0;
#pragma unroll
  for (int w = 0; w < WAVES; w++) total += s.part[w];
  __syncthreads();
  return total;
}

// The key at which a running sum over the visited keys, from the largest on, reaches
// `target` (0: goal(their sum)), digit by digit: visit(f) calls f(key, amount) for
// every key of this thread.  Returns the key; above: the sum of the larger keys;
// own: that of its equals.
template <class V, class Visit, class Goal>
__device__ __forceinline__ uint32_t find_key(Shared& s, V* bins, unsigned long long& target, Visit visit, Goal goal,
                                             unsigned long long& above, unsigned long long& own) {
  uint32_t prefix = 0;
  above = 0;
#pragma nounroll
  for (int low = 21, width = 11, done = 0;;) {  // digits of 11, 11 and 10 bits
    for (int i = threadIdx.x; i < BINS; i += THREADS) bins[i] = 0;
    __syncthreads();
    visit([&](uint32_t key, V amount) {
      if (done == 0 || key >> (32 - done) == prefix) atomicAdd(&bins[(key >> low) & ((1u << width) - 1)], amount);
    });
    __syncthreads();
    if (target == 0) target = goal(sum_bins(s, bins));
    find_bin(s, bins, target - above);
    prefix = prefix << width | (uint32_t)s.found[0];
    above += s.found[1];
    own = s.found[2];
    done += width;
    __syncthreads();
    if (low == 0) return prefix;
    width = low > 10 ? 11 : low;
    low -= width;
  }
}

template <class T>
__global__ void __launch_bounds__(THREADS) sample_rows(SampleArgs a) {
  constexpr int E = 16 / (int)sizeof(T);
  __shared__ Shared s;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t r = blockIdx.x;
  const T* row = (const T*)a.logits + r * a.vocab;
  const int steps = (a.vocab + THREADS * E - 1) / (THREADS * E);
  const double temperature = a.temperatures ? (double)a.temperatures[r] : a.temperature;
  const int64_t top_k = a.top_ks ? a.top_ks[r] : a.top_k;
  const double top_p = a.top_ps ? (double)a.top_ps[r] : a.top_p;
  const double asked = a.min_ps ? (double)a.min_ps[r] : a.min_p, min_p = asked <= 1.0 ? asked : 1.0;
  if (tid < 32) s.powers[tid] = exp2(tid * -0.03125);
  if (tid == 0) s.listed = 0;

  // the logits of tokens (step THREADS + thread) E .. + E as they lie in memory, NaN behind the last
  auto load = [&](int step, uint32_t (&w)[4]) {
    const int first = (step * THREADS + tid) * E;
    if (a.vector && first + E <= a.vocab) {
      const u32x4 v = global_load<u32x4>(row + first);
#pragma unroll
      for (int i = 0; i < 4; i++) w[i] = v[i];
    } else {
#pragma unroll
      for (int i = 0; i < 4; i++) {
        if constexpr (E == 4) {
          w[i] = first + i < a.vocab ? __float_as_uint(row[first + i]) : 0x7fc00000u;
        } else {
          w[i] = first + 2 * i < a.vocab ? row[first + 2 * i] : 0x7fc0u;
          w[i] |= (first + 2 * i + 1 < a.vocab ? row[first + 2 * i + 1] : 0x7fc0u) << 16;
        }
      }
    }
  };
  // all loads of the steps held are in flight together
  bool infinite = false;  // the row has +inf: those stand at 0, the others at -inf
  auto unpack = [&](const uint32_t (&w)[4], float (&v)[E]) {
#pragma unroll
    for (int e = 0; e < E; e++) {
      if constexpr (E == 4) v[e] = __uint_as_float(w[e]);
      else v[e] = __uint_as_float(e & 1 ? w[e >> 1] & 0xffff0000u : w[e >> 1] << 16);
    }
    if (infinite) {
#pragma unroll
      for (int e = 0; e < E; e++) v[e] = v[e] == INFINITY ? 0.f : -INFINITY;
    }
  };
  float largest[2] = {-INFINITY, -INFINITY};  // two maxima of each thread
  u32x32 held0, held1, held2, held3;
#pragma unroll
  for (int step = 0; step < HELD; step++) {
    uint32_t w[4] = {0xffc0ffc0u, 0xffc0ffc0u, 0xffc0ffc0u, 0xffc0ffc0u};  // NaN
    if (step < steps) load(step, w);
    float v[E];
    unpack(w, v);
#pragma unroll
    for (int e = 0; e < E; e++) largest[e & 1] = fmaxf(largest[e & 1], v[e]);
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const int at = 4 * (step % SPAN) + i;
      if (step < SPAN) held0[at] = w[i];
      else if (step < 2 * SPAN) held1[at] = w[i];
      else if (step < 3 * SPAN) held2[at] = w[i];
      else held3[at] = w[i];
    }
  }
  // f(step, words) for every step; those not held are loaded one step ahead
  auto each_word = [&](auto f) {
    uint32_t next[4] = {0u, 0u, 0u, 0u};
#pragma nounroll
    for (int step = 0; step < steps; step++) {
      uint32_t w[4];
      const int i = 4 * (step % SPAN);
      if (step < SPAN) w[0] = held0[i], w[1] = held0[i + 1], w[2] = held0[i + 2], w[3] = held0[i + 3];
      else if (step < 2 * SPAN) w[0] = held1[i], w[1] = held1[i + 1], w[2] = held1[i + 2], w[3] = held1[i + 3];
      else if (step < 3 * SPAN) w[0] = held2[i], w[1] = held2[i + 1], w[2] = held2[i + 2], w[3] = held2[i + 3];
      else if (step < HELD) w[0] = held3[i], w[1] = held3[i + 1], w[2] = held3[i + 2], w[3] = held3[i + 3];
      else w[0] = next[0], w[1] = next[1], w[2] = next[2], w[3] = next[3];
      if (step + 1 >= HELD && step + 1 < steps) load(step + 1, next);
      f(step, w);
    }
  };
  auto each = [&](auto f) {  // f(step, logits)
    each_word([&](int step, const uint32_t (&w)[4]) {
      float v[E];
      unpack(w, v);
      f(step, v);
    });
  };

  // ---- the largest logit
  for (int step = HELD; step < steps; step++) {
    uint32_t w[4];
    float v[E];
    load(step, w);
    unpack(w, v);
#pragma unroll
    for (int e = 0; e < E; e++) largest[e & 1] = fmaxf(largest[e & 1], v[e]);
  }
  float top = fmaxf(largest[0], largest[1]);
#pragma unroll
  for (int o = 32; o; o >>= 1) top = fmaxf(top, __shfl_xor(top, o));
  if (lane == 0) s.part[wave] = __float_as_uint(top);
  __syncthreads();
#pragma unroll
  for (int w = 0; w < WAVES; w++) top = fmaxf(top, __uint_as_float((uint32_t)s.part[w]));
  __syncthreads();
  if (top == -INFINITY) {
    if (tid == 0) a.tokens[r] = -1, a.probabilities[r] = 0.f;
    return;
  }
  if (!(temperature > 0.0)) {  // its lowest index
    uint32_t at = 0xffffffffu;
    each([&](int step, const float (&v)[E]) {
#pragma unroll
      for (int e = E - 1; e >= 0; e--) {
        const uint32_t i = (uint32_t)(step * THREADS + tid) * E + e;
        if (v[e] == top && i < at) at = i;
      }
    });
#pragma unroll
    for (int o = 32; o; o >>= 1) {
      const uint32_t other = __shfl_xor(at, o);
      at = other < at ? other : at;
    }
    if (lane == 0) s.part[wave] = at;
    __syncthreads();
    for (int w = 0; w < WAVES; w++) at = (uint32_t)s.part[w] < at ? (uint32_t)s.part[w] : at;
    if (tid == 0) a.tokens[r] = at, a.probabilities[r] = 1.f;
    return;
  }
  if (top == INFINITY) {
    infinite = true;
    top = 0.f;
#pragma unroll
    for (int i = 0; i < 2; i++) largest[i] = largest[i] == INFINITY ? 0.f : -INFINITY;
  }
  const Weigh weigh = {s.powers, (double)top, fmin(46.166241308446829 / temperature, 1e300)};  // 32 log2(e)
  const double unit = (double)(1ull << a.fraction);
  auto units = [&](double w) -> unsigned long long {  // w unit, rounded: at most 2^45
    return (unsigned long long)__double_as_longlong(fma(w, unit, 4503599627370496.0)) & 0xfffffffffffffull;
  };
  // the smallest logits that weigh something (2^-100 and min_p), and anything in a bin
  if (wave == 0) {
    const float least = least_of(top, [&](float l) { return weigh.behind(l) < 3200.0 && !(weigh(l) < min_p); });
    if (lane == 0) s.bound[0] = least;
  } else if (wave == 1) {
    const float least = least_of(top, [&](float l) { return weigh.behind(l) < 32.0 * (a.fraction + 1); });
    if (lane == 0) s.bound[1] = least;
  }
  __syncthreads();
  const float lightest = s.bound[0], binned = s.bound[1];

  // ---- the threshold: logits above it are kept, and `keep` of the `tied` on it
  float threshold = -INFINITY;
  unsigned long long keep = 0, tied = 0;
  const bool by_count = top_k > 0 && top_k < a.vocab, by_mass = top_p < 1.0;
  // the logits that the search is left with: from `low` on, below `high` (or all)
  float low = -INFINITY, high = 0.f;
  bool open = true, listed = false;
  unsigned long long target = 0, over = 0;  // of weights: what the prefix has to hold, and what lies above `high`
  auto target_of = [&](unsigned long long total) -> unsigned long long {
    const double wanted = ceil(top_p * (double)total);
    const unsigned long long least = wanted < 1.0 ? 1ull : (unsigned long long)wanted;
    return least < total ? least : total;
  };
  // bf16: the logits of each number are counted, and the threshold is a number
  bool counted = false;
  Window window = {1};
  if constexpr (E == 8) {
    const uint32_t widest = __float_as_uint(fmaxf(fabsf(top), fabsf(lightest))) >> 23 & 0xff;
    window.lo = (int)(widest < 20 ? 1 : (widest - 19) << 7);
    if (!infinite && (by_count || by_mass)) {
      for (int i = tid; i < ENTRIES; i += THREADS) s.numbers[i] = 0;
      __syncthreads();
      each_word([&](int, const uint32_t (&w)[4]) {
        uint32_t small = 0;
        s16x2 at[4];
#pragma unroll
        for (int i = 0; i < 4; i++) at[i] = window.entries(w[i], small);
#pragma unroll
        for (int i = 0; i < 4; i++) atomicAdd(&s.numbers[at[i][0]], 1u), atomicAdd(&s.numbers[at[i][1]], 1u);
        if (!__any(small & 0x80008000u)) return;
        float v[E];  // those below the window one by one into the list
        unpack(w, v);
#pragma unroll
        for (int e = 0; e < E; e++) {
          const bool in = (at[e >> 1][e & 1] == MAGNITUDES + 1 || at[e >> 1][e & 1] == MAGNITUDES + 2) && v[e] == v[e];
          const unsigned long long lanes = __ballot(in);
          if (!lanes) continue;
          uint32_t place = 0;
          if (lane == 0) place = atomicAdd(&s.listed, (uint32_t)__popcll(lanes));
          place = __shfl(place, 0) + (uint32_t)__popcll(lanes & ((1ull << lane) - 1));
          if (in && place < LIST) s.list[place] = v[e];
        }
      });
      __syncthreads();
      const int smaller = (int)s.listed;
      counted = smaller <= LIST;
      int entry = 0;
      if (counted && by_count) {
        // (a NaN's sign may put it above the window: it is no number)
        find_entry(s, [&](int i) -> unsigned long long { return i < ENTRIES - 1 ? s.numbers[i] : 0; },
                   (unsigned long long)top_k, [](unsigned long long n) { return n; });
        entry = (int)s.found[0];
        counted = window.holds(entry);
        tied = s.numbers[entry];
        keep = (unsigned long long)top_k - s.found[1];
        if (keep > tied) keep = tied;
        threshold = window.value(entry);
      }
      if (counted && by_mass) {
        // the weights of the numbers below the window, as one sum
        unsigned long long sum = 0;
        for (int i = tid; i < smaller; i += THREADS) sum += s.list[i] >= binned ? units(weigh(s.list[i])) : 0;
        sum = wave_sum(sum);
        __syncthreads();
        if (lane == 63) s.part[wave] = sum;
        __syncthreads();
        sum = 0;
        for (int w = 0; w < WAVES; w++) sum += s.part[w];
        __syncthreads();
        const int first = entry;
        const unsigned long long kept_there = keep;
        find_entry(s, [&](int i) -> unsigned long long {
          if (i < first) return 0;
          if (i == MAGNITUDES + 2) return sum;
          if (!window.holds(i)) return 0;
          const float l = window.value(i);
          const unsigned long long n = by_count && i == first ? kept_there : s.numbers[i];
          return n && l >= binned ? n * units(weigh(l)) : 0;
        }, 0, target_of);
        entry = (int)s.found[0];
        counted = window.holds(entry);
        if (counted) {
          threshold = window.value(entry);
          const unsigned long long one = units(weigh(threshold));
          keep = (s.found[3] - s.found[1] + one - 1) / one;
          tied = s.numbers[entry];
        }
      }
      __syncthreads();
      if (!counted) {  // it lies below the window (or too many do): found as fp32's is
        if (tid == 0) s.listed = 0;
        threshold = -INFINITY, keep = tied = 0;
        __syncthreads();
      }
    }
  }
  if (by_count && !counted) {
    // a bound that top_k logits reach: one that as many threads' maxima do
    if (a.vocab > LIST && top_k <= THREADS) {
      s.list[tid] = largest[0];
      s.list[THREADS + tid] = largest[1];
      __syncthreads();
      if (wave == 0) {
        uint32_t k[2 * WAVES], least = 0, most = key_of(top) + 1;
#pragma unroll
        for (int i = 0; i < 2 * WAVES; i++) k[i] = key_of(s.list[64 * i + lane]);
        while (most - least > 1) {  // least: reached by top_k maxima or more; most: by fewer
          const uint32_t mid = least + (most - least) / 2;
          int n = 0;
#pragma unroll
          for (int i = 0; i < 2 * WAVES; i++) n += __popcll(__ballot(k[i] >= mid));
          if (n >= top_k) least = mid;
          else most = mid;
          if (n >= top_k && n <= top_k + top_k / 4 + 8) break;
        }
        if (lane == 0) s.bound[2] = least <= key_of(-INFINITY) ? -INFINITY : value_of(least);
      }
      __syncthreads();
      low = s.bound[2];
    }
  } else if (by_mass && !counted) {
    for (int i = tid; i < BINS; i += THREADS) s.masses[i] = 0;
    __syncthreads();
    each([&](int, const float (&v)[E]) {
      int n[E];
      unsigned long long amount[E];
#pragma unroll
      for (int e = 0; e < E; e++) amount[e] = units(weigh(v[e], n[e]));
#pragma unroll
      for (int e = 0; e < E; e++)
        if (v[e] >= binned) atomicAdd(&s.masses[BINS - 1 - n[e]], amount[e]);
    });
    __syncthreads();
    target = target_of(sum_bins(s, s.masses));
    find_bin(s, s.masses, target);
    const int bin = BINS - 1 - (int)s.found[0];
    over = s.found[1];
    // the smallest logits of this bin and of the one above it
    if (wave < 2) {
      const double edge = bin - wave;
      const float least = least_of(top, [&](float l) { return weigh.behind(l) + ROUND - ROUND <= edge; });
      if (lane == 0) s.bound[2 + wave] = least;
    }
    __syncthreads();
    low = fmaxf(s.bound[2], binned), high = s.bound[3], open = bin == 0;
  }
  // these logits into the list, if they fit
  if (!counted && (by_count ? a.vocab <= LIST || top_k <= THREADS : by_mass)) {
    const float end = open ? INFINITY : high;  // (no logit here is +inf)
    each([&](int, const float (&v)[E]) {
      bool some = false;
#pragma unroll
      for (int e = 0; e < E; e++) some |= v[e] >= low && v[e] < end;
      if (!__any(some)) return;
#pragma unroll
      for (int e = 0; e < E; e++) {
        const bool in = v[e] >= low && v[e] < end;
        const unsigned long long lanes = __ballot(in);
        if (!lanes) continue;
        uint32_t at = 0;
        if (lane == 0) at = atomicAdd(&s.listed, (uint32_t)__popcll(lanes));
        at = __shfl(at, 0) + (uint32_t)__popcll(lanes & ((1ull << lane) - 1));
        if (in && at < LIST) s.list[at] = v[e];
      }
    });
    __syncthreads();
    listed = s.listed <= LIST;
  }
  // f(logit) for this thread's logits of the search
  auto visit = [&](auto f) {
    if (listed) {
      const int n = (int)s.listed;
      for (int i = tid; i < n; i += THREADS) f(s.list[i]);
    } else {
      each([&](int, const float (&v)[E]) {
#pragma unroll
        for (int e = 0; e < E; e++)
          if (v[e] >= low && (open || v[e] < high)) f(v[e]);
      });
    }
  };
  const int few = listed ? (int)s.listed : 0;
  if (few > 0 && few <= FEW) {
    // each logit of a short list against all of them
    const float l = tid < few ? s.list[tid] : -INFINITY;
    const unsigned long long amount = by_mass && tid < few && l >= binned ? units(weigh(l)) : 0;
    if (tid < FEW) s.masses[tid] = amount;
    if (tid < 4 && few + tid < LIST) s.list[few + tid] = NAN;
    __syncthreads();
    unsigned long long heavier = 0;
    int larger = 0, equal = 0;
    if (wave * 64 < few) {
      for (int j = 0; j < few; j += 2) {
        const float m0 = s.list[j], m1 = s.list[j + 1];
        const unsigned long long w0 = s.masses[j], w1 = s.masses[j + 1];
        larger += (m0 > l) + (m1 > l);
        equal += (m0 == l) + (m1 == l);
        heavier += (m0 > l ? w0 : 0) + (m1 > l ? w1 : 0);
      }
    }
    unsigned long long each_one = amount, goal = target - over;
    if (by_count) {
      const int wanted = (int)(top_k < few ? top_k : few);
      if (tid < few && larger < wanted && larger + equal >= wanted)  // those on the threshold, which agree
        s.found[0] = __float_as_uint(l), s.found[1] = wanted - larger, s.found[2] = equal, s.found[3] = heavier + amount * (unsigned long long)(wanted - larger);
      __syncthreads();
      threshold = __uint_as_float((uint32_t)s.found[0]);
      keep = s.found[1], tied = s.found[2];
      if (by_mass) goal = target_of(s.found[3]);
      __syncthreads();
    }
    if (by_mass) {
      const unsigned long long held = by_count && l == threshold ? keep : (unsigned long long)equal;
      if (tid < few && l >= threshold && heavier < goal && heavier + held * each_one >= goal)
        s.found[0] = __float_as_uint(l), s.found[1] = (goal - heavier + each_one - 1) / each_one, s.found[2] = equal;
      __syncthreads();
      threshold = __uint_as_float((uint32_t)s.found[0]);
      keep = s.found[1], tied = s.found[2];
    }
  } else if (!counted && (by_count || by_mass)) {
    if (by_count) {
      unsigned long long above, wanted = 0;
      auto goal = [&](unsigned long long n) { return (unsigned long long)top_k < n ? (unsigned long long)top_k : n; };
      const uint32_t key = find_key(s, s.counts, wanted, [&](auto f) { visit([&](float l) { f(key_of(l), 1u); }); }, goal,
                                    above, tied);
      threshold = value_of(key);
      keep = (unsigned long long)top_k - above;
      if (keep > tied) keep = tied;  // fewer numbers than top_k
      low = value_of(key + 1);       // for what lies above
    }
    if (by_mass) {
      unsigned long long above, own;
      target -= over;
      const uint32_t key = find_key(s, s.masses, target, [&](auto f) {
        visit([&](float l) {
          if (l >= low && l >= binned) f(key_of(l), units(weigh(l)));
        });
        // and what top_k keeps of its own threshold
        if (by_count && tid == 0 && threshold >= binned) f(key_of(threshold), keep * units(weigh(threshold)));
      }, target_of, above, own);
      const float l = value_of(key);
      const unsigned long long each_one = units(weigh(l));  // the tokens on a threshold weigh the same
      if (!by_count || l > threshold) tied = own / each_one;
      keep = (target - above + each_one - 1) / each_one;
      threshold = l;
    }
  }
  if (threshold < lightest) threshold = lightest, keep = tied = 0;

  // Where tokens on the threshold are left out (`cut`), a step's wave sums the weights above it and counts those
  // on it; what it keeps of them follows from the counts before it.
  const bool cut = keep < tied;
  const int slots = steps * WAVES;
  const double edge = cut ? weigh(threshold) : 0.0;
  __syncthreads();

  // the weights of this thread's tokens of a step above the threshold (and on it, where none is cut), 0 for others,
  // and how many of the wave's lie on a cut one; false where there are neither
  auto kept = [&](const float (&v)[E], double (&w)[E], uint32_t& on) -> bool {
    float most = v[0];
#pragma unroll
    for (int e = 1; e < E; e++) most = fmaxf(most, v[e]);
    if (!__any(most >= threshold)) return false;
    if (cut) {
#pragma unroll
      for (int e = 0; e < E; e++) on += (uint32_t)__popcll(__ballot(v[e] == threshold));
    }
#pragma unroll
    for (int e = 0; e < E; e++) w[e] = weigh(v[e]);
#pragma unroll
    for (int e = 0; e < E; e++) w[e] = (cut ? v[e] > threshold : v[e] >= threshold) ? w[e] : 0.0;
    return true;
  };

  // ---- their sums, step by step and wave by wave (the order of indices)
  if (E == 8 && !infinite) {
    if constexpr (E == 8) {
      // weights from the table, 0 for what is not kept; tokens below the window one by one
      for (int i = tid; i < ENTRIES; i += THREADS) {
        double x = 0.0;
        if (window.holds(i)) {
          const float l = window.value(i);
          if ((cut ? l > threshold : l >= threshold) && l <= top) x = weigh(l);
        }
        s.table[i] = x;
      }
      // the entry below which nothing is kept (a threshold that is no bf16 is cut towards 0; the zeros are equal)
      uint32_t unused = 0;
      const int entry = window.entries(__float_as_uint(threshold) >> 16, unused)[0];
      const int least = entry == MAGNITUDES + 2 ? MAGNITUDES + 1 : entry;
      const s16x2 edges = {(short)entry, (short)entry};
      __syncthreads();
      each_word([&](int step, const uint32_t (&w)[4]) {
        uint32_t small = 0, on = 0;
        s16x2 at[4];
#pragma unroll
        for (int i = 0; i < 4; i++) at[i] = window.entries(w[i], small);
        s16x2 most = __builtin_elementwise_max(__builtin_elementwise_max(at[0], at[1]), __builtin_elementwise_max(at[2], at[3]));
        double sum = 0.0;
        if (__any(most[0] >= least || most[1] >= least)) {
          if (__any(small & 0x80008000u)) {
            float v[E];
            double x[E];
            unpack(w, v);
            if (kept(v, x, on)) {
#pragma unroll
              for (int e = 0; e < E; e++) sum += x[e];
            }
          } else {
            double x[E];
#pragma unroll
            for (int e = 0; e < E; e++) x[e] = at[e >> 1][e & 1] >= least ? s.table[at[e >> 1][e & 1]] : 0.0;
#pragma unroll
            for (int e = 0; e < E; e++) sum += x[e];
            if (cut) {  // (the threshold is a number of the window, or the list gave it)
              uint32_t none = 0xffffffffu;
#pragma unroll
              for (int i = 0; i < 4; i++) {
                const uint32_t apart = __builtin_bit_cast(uint32_t, at[i] ^ edges);
                none &= ((apart & 0x7fff7fffu) + 0x7fff7fffu) | apart;
              }
              if (__any((none & 0x80008000u) != 0x80008000u)) {
                float v[E];
                unpack(w, v);
#pragma unroll
                for (int e = 0; e < E; e++) on += (uint32_t)__popcll(__ballot(v[e] == threshold));
              }
            }
          }
          sum = wave_sum(sum);
        }
        if (lane == 63) s.sums[step * WAVES + wave] = sum, s.ties[step * WAVES + wave] = on;
      });
    }
  } else {
    each([&](int step, const float (&v)[E]) {
      double w[E], sum = 0.0;
      uint32_t on = 0;
      if (kept(v, w, on)) {
#pragma unroll
        for (int e = 0; e < E; e++) sum += w[e];
        sum = wave_sum(sum);
      }
      if (lane == 63) s.sums[step * WAVES + wave] = sum, s.ties[step * WAVES + wave] = on;
    });
  }
  __syncthreads();
  if (wave == 0) {
    double before = 0.0;
    uint32_t ahead = 0;
    unsigned long long adds = 0;  // bit i0 / 64: this lane's sum there is not zero
    for (int i0 = 0; i0 < slots; i0 += 64) {
      const bool in = i0 + lane < slots;
      double run = in ? s.sums[i0 + lane] : 0.0;
      if (cut) {  // and the first `keep` of the tokens on the threshold
        const uint32_t n = in ? s.ties[i0 + lane] : 0;
        const uint32_t count = wave_scan(n);
        const uint32_t first = ahead + count - n;
        ahead += __shfl(count, 63);
        if (in) s.ties[i0 + lane] = first;
        if (first < keep) run += (double)(keep - first < n ? (uint32_t)keep - first : n) * edge;
      }
      if (run > 0.0) adds |= 1ull << (i0 / 64);
      run = wave_scan(run) + before;
      if (in) s.sums[i0 + lane] = run;
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
  double w[E] = {}, sum = 0.0;
  {
    uint32_t words[4];
    load(chosen / WAVES, words);
    float v[E];
    unpack(words, v);
    uint32_t on = 0;
    if (!kept(v, w, on)) return;
    if (cut) {
      unsigned long long rank = s.ties[chosen];
#pragma unroll
      for (int e = 0; e < E; e++) rank += __popcll(__ballot(v[e] == threshold) & ((1ull << lane) - 1));
#pragma unroll
      for (int e = 0; e < E; e++)
        if (v[e] == threshold && rank++ < keep) w[e] = edge;
    }
  }
#pragma unroll
  for (int e = 0; e < E; e++) sum += w[e];
  const double run = wave_scan(sum);
  const double base = chosen ? s.sums[chosen - 1] : 0.0;
  const unsigned long long past = __ballot(sum > 0.0 && base + run > goal), any = __ballot(sum > 0.0);
  const int owner = past ? __ffsll(past) - 1 : 63 - __clzll(any);
  if (lane != owner) return;
  double walk = base + run - sum, share = 0.0;
  int token = -1;
#pragma unroll
  for (int e = 0; e < E; e++) {
    if (w[e] > 0.0 && !(token >= 0 && walk > goal)) token = (chosen / WAVES * THREADS + tid) * E + e, share = w[e];
    walk += w[e];
  }
  a.tokens[r] = token;
  a.probabilities[r] = (float)(share / all);
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
                        62 - log2 < 45 ? 62 - log2 : 45};
  hipStream_t stream = (hipStream_t)stream_;
  if (dtype == BF16) hipLaunchKernelGGL(sample_rows<bf16_t>, dim3((unsigned)rows), dim3(THREADS), 0, stream, a);
  else hipLaunchKernelGGL(sample_rows<float>, dim3((unsigned)rows), dim3(THREADS), 0, stream, a);
  return (int)hipGetLastError();
}
